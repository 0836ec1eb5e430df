// Attention of a batch whose tokens share their first cells, and what every cell has been given by it.
//
//   s = q . k * scale,  p = exp(s - lse),  lse = log sum exp(s),  out = sum p v          over the cells [0, prompt) for every token, and behind them over the cells whose mask bit is set
//   mass[cell] <- decay * mass[cell] + sum over the tokens and heads that see it of p
//
// The query rows of a key head - tokens x its query heads - are one matrix against the prompt's keys.  A workgroup has 32 of these rows, or
// 128, and reads the keys for them; workgroups of the same keys follow each other, on one XCD where the keys' blocks divide by 8, so that memory gives a key once and the L2 the rest.  The cells behind the prompt differ from token to token: a workgroup takes one
// token's, listed from its mask, and reads no other, so that what stands in the others is without effect.  Scores are computed transposed (rows = cells): what a lane then holds - sixteen cells of one query - is, eight at a time, the
// operand of the product with the values, and the values come from LDS through its transposing load.
// Sums and statistics are fp32.  Products are fp16 x fp16 (exact in fp32); a weight is two fp16 values, rounded to nearest, the second one what the first leaves (23 bits; one alone, 11 bits, is 1.4e-4 off over 32000 cells).  fp16 ends at
// 2^-24, so weights are held relative to a power of two that follows them: up when they no longer fit, and down again behind a cell that took nearly all (px_weigh)
#include "ops_common.h"
#include "kernel_timing.h"
#include "wave_scan.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

typedef _Float16 px_half8 __attribute__((ext_vector_type(8)));
typedef _Float16 px_half2 __attribute__((ext_vector_type(2)));
typedef float px_f32x2 __attribute__((ext_vector_type(2)));
typedef short px_short4 __attribute__((ext_vector_type(4)));
typedef uint32_t px_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t px_u32x2 __attribute__((ext_vector_type(2)));
typedef float px_f32x16 __attribute__((ext_vector_type(16)));
typedef float px_f32x4 __attribute__((ext_vector_type(4)));

static __device__ __forceinline__ px_f32x16 px_mfma(px_u32x4 a, px_u32x4 b, px_f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(px_half8, a), __builtin_bit_cast(px_half8, b), c, 0, 0, 0); }
static __device__ __forceinline__ px_f32x16 px_zero() { return px_f32x16{ 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f }; }
// the cell of register i of a tile's scores, lane half g
static __device__ __forceinline__ int px_cell(int i, int g) { return 8 * (i >> 2) + 4 * g + (i & 3); }

// Bytes between rows in LDS.  Keys: an odd number of 16 bytes, so that the rows of a read of 16 bytes a lane lie apart.  Values: a transposing read takes 64 bytes of four rows for 32 lanes: 64 or 192 modulo 256
template <int DP> struct px_lds { static constexpr int K = 2 * DP + 16, V = (DP / 32) % 2 ? 2 * DP : 2 * DP + 64; };

// What weights are relative to, in powers of two.  (Tiles that are weighed twice: of scores of a deviation of up to two, and one cell far above them, one or two of a walk; of a deviation of four 8 of 32 and 10 of 100: 64 tokens of 64 / 8
// heads of 128 values, 32000 cells 126 us instead of 122, 100 tokens of 64 heads of 64 values, 4000 cells 37 instead of 32)
#define PX_MOST 65504.0f    /* a lane's weights of sixteen cells: fp16 holds them up to here, then it rises, */
#define PX_FULL 4096.0f     /* ... where weights are looked at, from here on: */
#define PX_TOP 4.0f         /* so that the tile's largest is 2^4, which leaves room for the next tiles', */
#define PX_ALONE 14.0f      /* or 2^14, where hardly another of the tile's is within */
#define PX_GAP 20.0f        /*    2^20 of it */
#define PX_FEW 4.0f         /* at the first tile it falls where they are this or less, and the largest less than a half, */
#define PX_LEAST 0.125f     /* at later ones where they are this or less */
#define PX_FALL 7.0f        /*    and the largest less than 2^-7, and rounded, at 2^-25, at 2^-18 of itself: so that it is 2^4 */
#define PX_HELD 60.0f       /* ... while the sums stay below 2^60: what is smaller beside them is lost to fp32 anyway */
#define PX_ROSE 4           /* rises of a walk that are looked behind */
#define PX_LIST 2048        /* cells of 64 words of a mask, a wave's */

// 32 queries of one key head, a column of the tile per lane, lanes l and l + 32 the same: their sums so far.  Of acc the outputs 32 j + px_cell(i, g); weights are 2^(score - m), l the sum of those of the lane's own cells (0: none)
template <int DP> struct px_sums { px_f32x16 acc[DP / 32]; float m, l; };
// of a walk over tiles: the next one, the one at which weights are looked at, rises that may still be looked behind
struct px_looks { int tile = 0, look = 0, spare = PX_ROSE; };
template <int DP> static __device__ __forceinline__ void px_start(px_sums<DP> & S) {
#pragma unroll
    for (int j = 0; j < DP / 32; j++) S.acc[j] = px_zero();
    S.m = S.l = 0.0f;
}

// scores of which the first `live` cells of the tile count
static __device__ __forceinline__ void px_only(px_f32x16 & s, int live, int g) {
#pragma unroll
    for (int i = 0; i < 16; i++) if (px_cell(i, g) >= live) s[i] = -INFINITY;
}

// a tile's weights, as operands of the products with the values: what a weight's first fp16 leaves in a second one
struct px_weights { px_u32x4 hi[2], lo[2]; };
static __device__ __forceinline__ void px_no_weights(px_weights & P) { for (int z = 0; z < 2; z++) P.hi[z] = P.lo[z] = px_u32x4{ 0, 0, 0, 0 }; }

// Of a tile's scores the weights and their sum; c = scale * log2(e).  S holds the products of the tiles before.
// What weights are relative to is not the largest score: any power of two is as good that keeps them within fp16, the sums are fp32.  It rises when a lane's weights no longer fit.  A cell far above the others would leave those only fp16's
// last bits, and where its values are small they are what the outputs are made of: so it falls again where a tile's weights are small.  That is looked for at tiles 0, 1, 5, 21, .. and behind the first rises, not at every tile: scores that
// are far apart from tile to tile would have it follow them up and down.  (One cell of 20 above 32000 others, its values zero: 7e-7 off; relative to the largest score, both halves cut off, 2.3e-4)
template <int DP> static __device__ __forceinline__ void px_weigh(px_sums<DP> & S, px_looks & W, px_weights & P, const px_f32x16 & s, float c) {
    float p[16], l = 0.0f, minus = -1.0f;
    asm("" : "+v"(minus));                                   // (unknown to the compiler: a - h would be a conversion and a subtraction, fma takes the fp16 as it is)
    auto weigh = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 16; i++) p[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -S.m));
        l = (((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]))) + (((p[8] + p[9]) + (p[10] + p[11])) + ((p[12] + p[13]) + (p[14] + p[15])));
#pragma unroll
        for (int z = 0; z < 2; z++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float a = p[8 * z + 2 * e], b = p[8 * z + 2 * e + 1];
                const px_half2 h = __builtin_convertvector((px_f32x2{ a, b }), px_half2);
                P.hi[z][e] = __builtin_bit_cast(uint32_t, h);
                P.lo[z][e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((px_f32x2{ fmaf((float) h[0], minus, a), fmaf((float) h[1], minus, b) }), px_half2));
            }
    };
    weigh();
    const bool looks = W.tile == W.look;
    const float most = looks ? PX_FULL : PX_MOST, least = W.tile == 0 ? PX_FEW : looks ? PX_LEAST : 0.0f;
    if (looks) W.look = 4 * W.tile + 1;
    if (__any(l > most || l <= least)) {
        float top = fmaxf(s[0], s[1]), next = fminf(s[0], s[1]);          // (next: one cell far above the others is not in it)
#pragma unroll
        for (int i = 2; i < 16; i += 2) { top = fmaxf(fmaxf(top, s[i]), s[i + 1]); next = fmaxf(next, fminf(s[i], s[i + 1])); }
        top = fmaxf(top, pi_partner<32>(top)) * c;
        next = fmaxf(next, pi_partner<32>(next)) * c;
        const float both = fmaxf(l, pi_partner<32>(l)), sum = S.l + pi_partner<32>(S.l);
        float m = S.m;
        const bool rises = both > most;
        if (rises) m = top - (top - next > PX_GAP ? PX_ALONE : PX_TOP);
        else if (both <= least && top < m - (W.tile == 0 ? 1.0f : PX_FALL) && top > -INFINITY) m = fmaxf(top - PX_TOP, m - PX_HELD + __builtin_amdgcn_logf(sum));
        if (W.spare > 0 && !looks && __any(rises)) { W.look = W.tile + 1; W.spare--; }
        if (looks && __any(top == -INFINITY)) W.look = W.tile + 1;        // (nothing to look at yet)
        const float f = sum == 0.0f ? 1.0f : __builtin_amdgcn_exp2f(S.m - m);
        S.m = m; S.l *= f;
#pragma unroll
        for (int j = 0; j < DP / 32; j++)
#pragma unroll
            for (int i = 0; i < 16; i++) S.acc[j][i] *= f;
        weigh();
    }
    S.l += l;
    W.tile++;
}

// the values' operand from rows of `stride` bytes in LDS: at = the wave's first row + px_value_at; sixteen lanes take four rows of sixteen values and each gets a column
static __device__ __forceinline__ int px_value_at(int lane, int stride) { return ((lane & 15) / 4 + 4 * (lane >> 5)) * stride + 32 * (lane >> 4 & 1) + 8 * (lane & 3); }
template <int STRIDE> static __device__ __forceinline__ px_u32x4 px_value(const uint8_t * at, int j, int z) {
    typedef __attribute__((address_space(3))) px_short4 lds4;
    const px_u32x2 a = __builtin_bit_cast(px_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *) (at + 16 * z * STRIDE + 64 * j)));
    const px_u32x2 b = __builtin_bit_cast(px_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *) (at + (16 * z + 8) * STRIDE + 64 * j)));
    return px_u32x4{ a[0], a[1], b[0], b[1] };
}

// the products of a tile's weights with its values, whose first row is px_value_at behind `at`
template <int DP, int VS> static __device__ __forceinline__ void px_products(px_sums<DP> & S, const px_weights & P, const uint8_t * at) {
#pragma unroll
    for (int j = 0; j < DP / 32; j++)
#pragma unroll
        for (int z = 0; z < 2; z++) {
            const px_u32x4 v = px_value<VS>(at, j, z);
            S.acc[j] = px_mfma(v, P.hi[z], S.acc[j]);
            S.acc[j] = px_mfma(v, P.lo[z], S.acc[j]);
        }
}

// n / d for n < 2^31 (a division by what only the arguments know is thirty instructions, and a kernel that runs for a few us waits for every line of code that it has not run yet: 80 clocks for 64 bytes)
struct px_div { uint32_t mul, shift; };
static px_div px_divide_by(uint32_t d) {
    uint32_t s = 0;
    while ((1ull << s) < d) s++;
    return { (uint32_t) (((1ull << (31 + s)) + d - 1) / d), 31 + s };
}
static __device__ __forceinline__ uint32_t px_quotient(uint32_t n, px_div d) { return (uint32_t) (((uint64_t) n * d.mul) >> d.shift); }

struct px_args {
    const uint16_t * q; int64_t q_stride;
    const uint16_t * k, * v; int64_t row;                    // a cell's values: all key heads
    const uint32_t * mask; const int32_t * dyn;
    float c;
    int dim, heads, kv, group, n_tok, prompt, n_kv;
    int row_blocks, prompt_parts, own_blocks, own_parts;     // of a key head's rows; parts that the prompt is cut into; blocks of 32 of a token's rows; parts of the cells behind it
    px_div by_group, by_kv, by_row_blocks, by_own_blocks, by_own_parts, by_parts, by_quads;
    int prompt_share, own_share;                             // cells, words of the mask of a part where the sizes are the arguments'
    bool wide, together;                                     // blocks of 128 rows; the prompt's workgroups take the own cells too
    float * parts_o; float2 * parts_ml;                      // [part][token][head][dim], [part][token][head] (maximum, sum)
    float * out; int64_t out_stride; float * lse;
};

// Outputs that are no finite numbers although the sum of the weights `l` is: a value that the token sees is infinite, and one of a weight's two halves was zero.  They are the sum of what is not finite among its values.
// o: the token's outputs of the head; from `d` on, every step-th four.  (Off the way: a thread reads the values of all cells, eight at a time - 1 token of 64 / 8
// heads of 128 values over 32000 cells, one of them infinite: 5.6 ms, 64 such tokens 17)
static __device__ __forceinline__ bool px_finite(float x) { return fabsf(x) < INFINITY; }
static __device__ __forceinline__ bool px_finite(px_f32x4 x) { return px_finite(x[0]) && px_finite(x[1]) && px_finite(x[2]) && px_finite(x[3]); }
static __device__ __forceinline__ void px_infinite(const px_args & A, float * o, int tok, int head, int d, int step) {
    const int n_kv = A.dyn ? max(0, min(A.dyn[1], A.n_kv)) : A.n_kv, prompt = min(A.dyn ? max(0, min(A.dyn[0], A.prompt)) : A.prompt, n_kv), n = A.mask ? n_kv : prompt;
    const uint32_t * mask = A.mask + (int64_t) tok * ((A.n_kv + 31) / 32);
    for (; d < A.dim; d += step) {
        px_f32x4 x = *(px_f32x4 *) (o + d), sum = { 0.0f, 0.0f, 0.0f, 0.0f };
        if (px_finite(x)) continue;
        const uint16_t * v = A.v + head / A.group * A.dim + d;
#pragma unroll 1
        for (int c0 = 0; c0 < n; c0 += 8) {
            px_u32x2 of[8];
#pragma unroll
            for (int i = 0; i < 8; i++) of[i] = *(const px_u32x2 *) (v + (int64_t) min(c0 + i, n - 1) * A.row);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int c = min(c0 + i, n - 1);
                const bool sees = c < prompt || (mask[c >> 5] >> (c & 31) & 1);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float y = (float) __builtin_bit_cast(_Float16, (uint16_t) (of[i][e >> 1] >> (16 * (e & 1))));
                    if (sees && !px_finite(y)) sum[e] += y;
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 4; e++) if (!px_finite(x[e]) && sum[e] != 0.0f) x[e] = sum[e];
        *(px_f32x4 *) (o + d) = x;
    }
}

// the sums of 32 rows of key head j from row0 on: part `part` of theirs, or the result where it is the only one
template <int DP> static __device__ __forceinline__ void px_leave(const px_args & A, px_sums<DP> & S, int part, int tok, int head, bool mine, int g) {
    const float l = S.l + pi_partner<32>(S.l);
    if (!mine) return;
    const bool last = A.prompt_parts + A.own_parts == 1;
    const int64_t r = (int64_t) tok * A.heads + head;
    float * o;
    float f = 1.0f;
    if (last) {
        o = A.out + (int64_t) tok * A.out_stride + (int64_t) head * A.dim;
        f = l == 0.0f ? 0.0f : 1.0f / l;
        if (g == 0 && A.lse) A.lse[r] = l == 0.0f ? -INFINITY : (S.m + __builtin_amdgcn_logf(l)) * 0.693147181f;
    } else {
        const int64_t at = (int64_t) part * A.n_tok * A.heads + r;
        o = A.parts_o + at * A.dim;
        if (g == 0) A.parts_ml[at] = make_float2(S.m, l);
        if (l == 0.0f) return;                               // (k_prefix_merge leaves such a part out)
    }
    auto leave = [&](auto whole) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < DP / 32; j++)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int d = 32 * j + px_cell(i, g);
                if (whole || d < A.dim) *(px_f32x4 *) (o + d) = px_f32x4{ S.acc[j][i] * f, S.acc[j][i + 1] * f, S.acc[j][i + 2] * f, S.acc[j][i + 3] * f };
            }
    };
    if (A.dim == DP) leave(std::true_type{}); else leave(std::false_type{});
    if (!last || !(l > 0.0f) || !px_finite(l)) return;
    float all = 0.0f;                                        // (no number, or 0)
#pragma unroll
    for (int j = 0; j < DP / 32; j++)
#pragma unroll
        for (int i = 0; i < 16; i++) all = fmaf(S.acc[j][i], 0.0f, all);
    if (all != 0.0f) px_infinite(A, o, tok, head, 4 * g, 8);
}

// values d .. d + 7 of a row of `dim`, zeros behind its end (read without a branch: behind one, a load is waited for where the branches meet)
static __device__ __forceinline__ px_u32x4 px_chunk(const uint16_t * row, int d, int dim) {
    const px_u32x4 x = *(const px_u32x4 *) (row + (d < dim ? d : 0));
    px_u32x4 y;
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = d < dim ? x[e] : 0u;
    return y;
}
template <int DP> static __device__ __forceinline__ void px_queries(const px_args & A, px_u32x4 (&q)[DP / 16], int tok, int head, int g) {
    const uint16_t * row = A.q + (int64_t) tok * A.q_stride + (int64_t) head * A.dim;
#pragma unroll
    for (int i = 0; i < DP / 16; i++) q[i] = px_chunk(row, 16 * i + 8 * g, A.dim);
}

// Many rows: a wave has 32 of the workgroup's 128, all walk the same cells, 32 at a time through a ring of four tiles in LDS.  Three tiles are in work at once, so that the matrix cores and the vector unit are: while the weights of tile t are
// made from its scores, the products of the weights of t - 1 with the values and of the keys of t + 1 with the queries run; tile t + 2 goes to LDS and t + 3 is on its way in registers
template <int DP> static __device__ __forceinline__ void px_wide(const px_args & A, uint8_t * lds, int kvh, int block, int part, int c0, int c1) {
    constexpr int KS = px_lds<DP>::K, VS = px_lds<DP>::V, TILE = 32 * (KS + VS), CH = DP / 8, N = (32 * CH + 255) / 256;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, g = lane >> 5, rows = A.n_tok * A.group, tiles = (c1 - c0 + 31) / 32;
    const int row = block * 128 + wave * 32 + n, at = min(row, rows - 1), tok = (int) px_quotient((uint32_t) at, A.by_group), head = kvh * A.group + at - tok * A.group;
    px_u32x4 q[DP / 16], kr[N], vr[N];
    px_queries<DP>(A, q, tok, head, g);
    px_sums<DP> S;
    px_start(S);
    const uint16_t * k = A.k + kvh * A.dim, * v = A.v + kvh * A.dim;
    // (a chunk past the head's end reads its first, and is not stored: zeros stand there, as in the queries - an infinity of the keys would make no number of them)
    auto in_head = [&](int i) __attribute__((always_inline)) { return min(i * 256 + tid, 32 * CH - 1) % CH * 8 < A.dim; };
    auto load = [&](int t) __attribute__((always_inline)) {
        const int64_t c = c0 + 32 * t;
        const uint16_t * kc = k + c * A.row, * vc = v + c * A.row;
        const int last = c1 - 1 - c0 - 32 * t;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int x = min(i * 256 + tid, 32 * CH - 1), d = x % CH * 8;
            const uint32_t o = (uint32_t) (last >= 31 ? x / CH : min(x / CH, last)) * (uint32_t) A.row + (uint32_t) (d < A.dim ? d : 0);
            kr[i] = *(const px_u32x4 *) (kc + o);
            vr[i] = *(const px_u32x4 *) (vc + o);
        }
    };
    auto store = [&](int t) __attribute__((always_inline)) {
        uint8_t * to = lds + (t & 3) * TILE;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int x = min(i * 256 + tid, 32 * CH - 1);
            if (!in_head(i)) continue;
            *(px_u32x4 *) (to + x / CH * KS + x % CH * 16) = kr[i];
            *(px_u32x4 *) (to + 32 * KS + x / CH * VS + x % CH * 16) = vr[i];
        }
    };
    if (A.dim < DP)
#pragma unroll 1
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int x = min(i * 256 + tid, 32 * CH - 1);
                if (!in_head(i)) *(px_u32x4 *) (lds + t * TILE + x / CH * KS + x % CH * 16) = *(px_u32x4 *) (lds + t * TILE + 32 * KS + x / CH * VS + x % CH * 16) = px_u32x4{ 0, 0, 0, 0 };
            }
    auto scores = [&](int t) __attribute__((always_inline)) {
        const uint8_t * kt = lds + (t & 3) * TILE + n * KS + 16 * g;
        px_f32x16 s = px_zero();
#pragma unroll
        for (int i = 0; i < DP / 16; i++) s = px_mfma(*(const px_u32x4 *) (kt + 32 * i), q[i], s);
        return s;
    };
    load(0);
#pragma unroll 1
    for (int t = 0; t < 2; t++) {                            // (code that runs once costs more than it does)
        if (t < tiles) store(t);
        if (t + 1 < tiles) load(t + 1);
    }
    __syncthreads();
    px_f32x16 s = scores(0);
    px_weights P;
    px_looks W;
    px_no_weights(P);
    const int value_at = 32 * KS + px_value_at(lane, VS);
    for (int t = 0; t < tiles; t++) {
        if (t > 0) __syncthreads();
        if (t + 2 < tiles) store(t + 2);
        if (t + 3 < tiles) load(t + 3);
        if (c0 + 32 * t + 32 > c1) px_only(s, c1 - c0 - 32 * t, g);
        // (of the first tile no weights: its own values times 0; behind the last one the scores of whatever stands there, for nobody)
        px_products<DP, VS>(S, P, lds + (max(t - 1, 0) & 3) * TILE + value_at);
        const px_f32x16 next = scores(t + 1);
        px_weigh<DP>(S, W, P, s, A.c);
        s = next;
    }
    px_products<DP, VS>(S, P, lds + (tiles - 1 & 3) * TILE + value_at);
    px_leave<DP>(A, S, part, tok, head, row < rows, g);
}

// Few rows, 32 of them: a wave walks the runs of 32 cells first, first + step, .. of `count`, the i-th at cell_of(i); sums go on in S.  Keys come as operands, values to a part of LDS that is the wave's
// own, so that no wave waits for another; the next run's are on their way meanwhile
template <int DP, class C> static __device__ __forceinline__ void px_walk(const px_args & A, px_sums<DP> & S, const px_u32x4 (&q)[DP / 16], uint8_t * mine, int kvh, int first, int step, int lane, int count, C && cell_of) {
    constexpr int VS = px_lds<DP>::V, CH = DP / 8, N = DP / 16;
    const int n = lane & 31, g = lane >> 5;
    const uint16_t * k = A.k + kvh * A.dim, * v = A.v + kvh * A.dim;
    px_u32x4 kr[N], vr[N];
    auto load = [&](int at) __attribute__((always_inline)) {
        const uint16_t * kc = k + (int64_t) cell_of(min(at + n, count - 1)) * A.row;
#pragma unroll
        for (int i = 0; i < N; i++) kr[i] = *(const px_u32x4 *) (kc + (16 * i + 8 * g < A.dim ? 16 * i + 8 * g : 0));
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int x = i * 64 + lane, d = x % CH * 8;
            vr[i] = *(const px_u32x4 *) (v + (int64_t) cell_of(min(at + x / CH, count - 1)) * A.row + (d < A.dim ? d : 0));
        }
    };
    if (first >= count) return;
    px_looks W;
    load(first);
    for (int at = first; at < count; at += step) {
        px_u32x4 kc[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            kc[i] = kr[i];
            const int x = i * 64 + lane;
            *(px_u32x4 *) (mine + x / CH * VS + x % CH * 16) = vr[i];
        }
        if (A.dim < DP)                                      // (as the queries there: an infinity of the keys' first values would make no number of them; the least that goes by DP is DP - 56)
#pragma unroll
            for (int i = N > 4 ? N - 4 : 0; i < N; i++) if (16 * i + 8 * g >= A.dim) kc[i] = px_u32x4{ 0, 0, 0, 0 };
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        if (at + step < count) load(at + step);
        const uint8_t * vt = mine + px_value_at(lane, VS);
        px_f32x16 s = px_zero();
#pragma unroll
        for (int i = 0; i < N; i++) s = px_mfma(kc[i], q[i], s);
        if (at + 32 > count) px_only(s, count - at, g);
        px_weights P;
        px_weigh<DP>(S, W, P, s, A.c);
        px_products<DP, VS>(S, P, vt);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// the sums of the four waves, of the same rows, put together in LDS by all of them and left as px_leave does; lds: 4 * DP * 128 bytes and 1 KB behind, no wave in its own part any more
template <int DP> static __device__ __forceinline__ void px_meet(const px_args & A, px_sums<DP> & S, uint8_t * lds, int wave, int lane, int part, int tok, int head, bool mine) {
    const int n = lane & 31, g = lane >> 5;
    float2 * const ml = (float2 *) (lds + 4 * DP * 128);
    const float own = S.l + pi_partner<32>(S.l);
    __syncthreads();
    if (g == 0) ml[wave * 32 + n] = make_float2(S.m, own);
    __syncthreads();
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) { const float2 x = ml[w * 32 + n]; if (x.y != 0.0f) m = fmaxf(m, x.x); }
#pragma unroll
    for (int w = 0; w < 4; w++) { const float2 x = ml[w * 32 + n]; if (x.y != 0.0f) l += x.y * __builtin_amdgcn_exp2f(x.x - m); }
    const bool last = A.prompt_parts + A.own_parts == 1;
    const float f = own == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(S.m - m) * (last ? 1.0f / l : 1.0f);
    px_f32x4 * const at = (px_f32x4 *) lds;                  // [4 j + i / 4][wave][lane]
#pragma unroll
    for (int j = 0; j < DP / 32; j++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) at[((4 * j + i / 4) * 4 + wave) * 64 + lane] = px_f32x4{ S.acc[j][i] * f, S.acc[j][i + 1] * f, S.acc[j][i + 2] * f, S.acc[j][i + 3] * f };
    __syncthreads();
    const int64_t r = (int64_t) tok * A.heads + head, to = (int64_t) part * A.n_tok * A.heads + r;
    if (wave == 0 && g == 0 && mine) {
        if (!last) A.parts_ml[to] = make_float2(m, l);
        else if (A.lse) A.lse[r] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * 0.693147181f;
    }
    if (!mine || (l == 0.0f && !last)) return;               // (k_prefix_merge leaves such a part out)
    float * o = last ? A.out + (int64_t) tok * A.out_stride + (int64_t) head * A.dim : A.parts_o + to * A.dim;
    bool odd = false;
#pragma unroll
    for (int k = 0; k < DP / 32; k++) {
        const int i = 4 * k + wave, d = 8 * i + 4 * g;
        const px_f32x4 a = at[(i * 4) * 64 + lane], b = at[(i * 4 + 1) * 64 + lane], c = at[(i * 4 + 2) * 64 + lane], e = at[(i * 4 + 3) * 64 + lane];
        if (d >= A.dim) continue;
        const px_f32x4 x = (a + b) + (c + e);
        *(px_f32x4 *) (o + d) = x;
        odd |= !px_finite(x);
    }
    if (odd && last && px_finite(l)) px_infinite(A, o, tok, head, 8 * wave + 4 * g, 32);
}

// part `part` of n things in shares of `share`
static __device__ __forceinline__ void px_share(int n, int share, int part, int & from, int & to) { from = (int) min((int64_t) n, (int64_t) part * share); to = (int) min((int64_t) n, (int64_t) from + share); }
// a share of n things in whole runs of `run`, so that `parts` of them are all
static __host__ __device__ __forceinline__ int px_share_of(int n, int run, int parts) { const uint32_t runs = ((uint32_t) n + run - 1) / run; return (int) ((runs + parts - 1) / parts) * run; }

// Many rows and cells are bound by the matrix cores and the vector unit in turns (64 tokens of 64 / 8 heads of 128 values, 32000 cells: 120 us, 101 GFLOP with the weights' second halves, 840 TFLOP/s; of the clocks 45 % matrix, 40 % vector:
// the registers of two waves are full, so little of one runs under the other); keys of their own for every head by the caches' rows (24 tokens, 2047 cells, 51 MB: 15 us, 3.4 TB/s); what lies between by the chain of a workgroup's few tiles
// (16 tokens of 64 / 8 heads, 4000 cells, 22 MB: 15 us - 3 until the first rows are there, 5 for four runs of 32 cells a wave, 2 to meet; a token of 32 / 4 heads of 64 values, 513 cells: 8 us)
// (Registers for four, three, two workgroups a compute unit are asked for: heads of 64 values otherwise take 170 and two fit, 100 tokens of 64 heads of 64 values, 4000 cells 36 us instead of 32)
template <int DP, bool WIDE> __global__ void __launch_bounds__(256, DP <= 32 ? 4 : DP <= 64 ? 3 : DP <= 128 ? 2 : 1) k_prefix_attention(const px_args A, const int32_t * __restrict__ abort_w) {
    if (pi_aborted(abort_w, 5)) return;                      // (what a wave takes from LDS as an index, it has put there itself)
    constexpr int NARROW = 4 * (32 * px_lds<DP>::V + 2 * PX_LIST), MEET = 4 * DP * 128 + 1024, WIDE_B = WIDE ? 4 * 32 * (px_lds<DP>::K + px_lds<DP>::V) : MEET;
    __shared__ __attribute__((aligned(16))) uint8_t lds[NARROW > WIDE_B ? NARROW : WIDE_B];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, g = lane >> 5;
    const int n_kv = A.dyn ? max(0, min(A.dyn[1], A.n_kv)) : A.n_kv, prompt = min(A.dyn ? max(0, min(A.dyn[0], A.prompt)) : A.prompt, n_kv);
    const uint32_t pairs = (uint32_t) A.kv * A.prompt_parts, prompt_blocks = pairs * A.row_blocks;
    px_u32x4 q[DP / 16];
    px_sums<DP> S;
    uint8_t * mine = lds + wave * 32 * px_lds<DP>::V;
    const bool shared = blockIdx.x < prompt_blocks;
    int part, kvh, tok, head, in, rows = A.group;              // in: the lane's row, of `rows`
    uint32_t whose = 0;                                        // (the token whose own cells are walked)
    if (shared) {
        // the blocks of rows that read the same keys follow each other on one XCD (a workgroup's is its number modulo 8)
        const uint32_t b = blockIdx.x, eights = pairs % 8 == 0, of = eights ? b >> 3 : b, by = px_quotient(of, A.by_row_blocks), block = of - by * A.row_blocks, pair = eights ? by * 8 + (b & 7) : by;
        part = (int) px_quotient(pair, A.by_kv); kvh = (int) pair - part * A.kv;
        int c0, c1;
        px_share(prompt, A.dyn ? px_share_of(prompt, 32, A.prompt_parts) : A.prompt_share, part, c0, c1);
        rows = A.n_tok * A.group;
        if constexpr (WIDE) {
            if (c0 >= c1) {                                  // (fewer cells than there may be)
                px_start(S);
                in = block * 128 + wave * 32 + n;
                const int at = min(in, rows - 1);
                tok = (int) px_quotient((uint32_t) at, A.by_group);
                px_leave<DP>(A, S, part, tok, kvh * A.group + at - tok * A.group, in < rows, g);
            } else px_wide<DP>(A, lds, kvh, (int) block, part, c0, c1);
            return;
        } else {
            in = block * 32 + n;
            const int at = min(in, rows - 1);
            tok = (int) px_quotient((uint32_t) at, A.by_group); head = kvh * A.group + at - tok * A.group;
            px_queries<DP>(A, q, tok, head, g);
            px_start(S);
            px_walk<DP>(A, S, q, mine, kvh, 32 * wave, 128, lane, c1 - c0, [&](int i) __attribute__((always_inline)) { return c0 + i; });
        }
    }
    // A token's own cells: a wave takes 32 of the query heads of one key head, and 64 words of the mask at a time; or, of a single token behind a short prompt, the four waves of the prompt's workgroup, every fourth 32 cells each
    const int words = (A.n_kv + 31) / 32, w0 = prompt / 32, w_all = max(0, (n_kv + 31) / 32 - w0);
    uint16_t * list = (uint16_t *) (lds + 4 * 32 * px_lds<DP>::V) + wave * PX_LIST;
    int from = 0, to = A.together ? w_all : 0;
    if (!shared) {
        const uint32_t unit = (blockIdx.x - prompt_blocks) * 4 + __builtin_amdgcn_readfirstlane(wave);
        const uint32_t a = px_quotient(unit, A.by_kv), c = px_quotient(a, A.by_own_blocks);
        whose = px_quotient(c, A.by_own_parts);
        if (whose >= (uint32_t) A.n_tok) return;
        kvh = (int) (unit - a * A.kv); tok = (int) whose; part = (int) (c - whose * A.own_parts); in = (int) (a - c * A.own_blocks) * 32 + n; head = kvh * A.group + min(in, A.group - 1);
        px_share(w_all, A.dyn ? px_share_of(w_all, 2, A.own_parts) : A.own_share, part, from, to);
        part += A.prompt_parts;
        px_queries<DP>(A, q, tok, head, g);
        px_start(S);
    }
    for (int w = from; w < to; w += 64) {
        const int at = w0 + min(w + lane, to - 1);
        uint32_t bits = A.mask[(int64_t) whose * words + at];
        if (w + lane >= to) bits = 0;
        if (32 * at < prompt) bits &= ~0u << (prompt - 32 * at);                // (prompt - 32 * at < 32: at >= prompt / 32)
        if (n_kv - 32 * at < 32) bits &= (1u << (n_kv - 32 * at)) - 1;
        const int upto = (int) pi_wave_scan((uint32_t) __popc(bits)), count = __builtin_amdgcn_readlane(upto, 63);
        int before = upto - __popc(bits);
        for (uint32_t left = bits; left; left &= left - 1) list[before++] = (uint16_t) (32 * lane + __builtin_ctz(left));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const int first = 32 * (w0 + w);
        px_walk<DP>(A, S, q, mine, kvh, shared ? 32 * wave : 0, shared ? 128 : 32, lane, count, [&](int i) __attribute__((always_inline)) { return first + list[i]; });
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    if (shared) px_meet<DP>(A, S, lds, wave, lane, part, tok, head, in < rows);
    else px_leave<DP>(A, S, part, tok, head, in < rows, g);
}

#define PX_PARTS 1088       /* what k_prefix_merge has room for; the prompt takes two of a compute unit's at most */
// The parts' sums over their joint maximum.  Four of a row's values to a thread and about every `groups`-th part, the threads of a row meet in LDS: with a wave per row and its parts one after the other the loads' latency was all the
// time (4096 rows of 17 parts: 24.2 us; 1024 of 17: 20.8).  Bound by the parts' rows (4096 rows of 17: 12.0 us, 38 MB at 3.2 TB/s; 768 of 9: 4.0)
__global__ void __launch_bounds__(256) k_prefix_merge(const px_args A, int parts, int log_groups, int rows_here, const int32_t * __restrict__ abort_w) {
    if (pi_aborted(abort_w, 5)) return;
    __shared__ float2 ml[PX_PARTS];                         // (512 of them at most where the workgroup has more than one row)
    __shared__ px_f32x4 sums[256];
    __shared__ float ls[256];
    const int tid = threadIdx.x, quads = A.dim / 4, at = (int) px_quotient((uint32_t) tid, A.by_quads), d = 4 * (tid - at * quads), mine = at >> log_groups, groups = 1 << log_groups, grp = at & (groups - 1);
    const int64_t rows = (int64_t) A.n_tok * A.heads, r0 = (int64_t) blockIdx.x * rows_here;
    const bool on = mine < rows_here && r0 + mine < rows;
    const float * from = A.parts_o + min(r0 + mine, rows - 1) * A.dim + d;
    const int64_t step = rows * A.dim;
    px_f32x4 x[4];
    auto load = [&](int p) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = *(const px_f32x4 *) (from + min(p + i * groups, parts - 1) * step);
    };
    if (parts > 0) load(grp);
    for (int i = tid; i < rows_here * parts; i += 256) {
        const int of = (int) px_quotient((uint32_t) i, A.by_parts);
        float2 v = A.parts_ml[(i - of * parts) * rows + min(r0 + of, rows - 1)];
        if (v.y == 0.0f) v.x = -INFINITY;                    // (a part without a cell: its outputs are not there)
        ml[i] = v;
    }
    __syncthreads();
    float m = -INFINITY, l = 0.0f;
    px_f32x4 o = { 0.0f, 0.0f, 0.0f, 0.0f };
    if (on) {
        const float2 * of = ml + mine * parts;
#pragma unroll 1
        for (int p = 0; p < parts; p += 8)
#pragma unroll
            for (int i = 0; i < 8; i++) m = fmaxf(m, of[min(p + i, parts - 1)].x);
        const float from_m = m == -INFINITY ? 0.0f : m;
        for (int p = grp; p < parts; p += 4 * groups) {
            if (p != grp) load(p);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float2 v = of[min(p + i * groups, parts - 1)];
                if (p + i * groups >= parts) v.y = 0.0f;
                const float f = __builtin_amdgcn_exp2f(v.x - from_m);
                l += v.y * f;
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] += v.y == 0.0f ? 0.0f : x[i][e] * f;
            }
        }
    }
    if (groups > 1) {
        sums[tid] = o; ls[tid] = l;
        __syncthreads();
        if (grp != 0 || !on) return;
        for (int i = 1; i < groups; i++) { o += sums[tid + i * quads]; l += ls[tid + i * quads]; }
    }
    if (!on) return;
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
    const int64_t r = r0 + mine;
    float * to = A.out + r / A.heads * A.out_stride + r % A.heads * A.dim;
    o *= f;
    *(px_f32x4 *) (to + d) = o;
    if (!px_finite(o) && px_finite(l)) px_infinite(A, to, (int) (r / A.heads), (int) (r % A.heads), d, A.dim);
    if (d == 0 && A.lse) A.lse[r] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * 0.693147181f;
}

// ---- how the work is cut ---------------------------------------------------------------------------------------------------------------------------------------------------------------
// device: the sizes are the device's, which may leave cells behind the prompt where the arguments leave none
static void px_plan(px_args & A, bool device) {
    const int rows = A.n_tok * A.group, target = 2 * pi_cu_count();
    A.own_blocks = (A.group + 31) / 32;
    const int64_t own = (int64_t) A.n_tok * A.kv * A.own_blocks, narrow = (int64_t) A.kv * ((rows + 31) / 32);
    // More than 64 rows go by 128, four waves past the same tiles, where there is work for it - scores times values from 2^31 on (64 tokens of 64 / 8 heads of 128 values: 8000 cells 46 us, by 32 rows 56; 4000 cells 34 and 34; 2000 cells
    // 30 and 25) - or where blocks of 32 rows and the tokens' own cells would be more workgroups than run at once (100 tokens of 32 heads with keys of their own, 600 cells: 21 us and 24; 200 of 64 / 8 heads, 1000 cells: 28 and 34)
    A.wide = rows > 64 && (narrow + own / 4 > target || (double) A.kv * rows * A.prompt * A.dim > 0x1p31);
    A.row_blocks = A.wide ? (rows + 127) / 128 : (rows + 31) / 32;
    const int64_t units = (int64_t) A.kv * A.row_blocks;
    const int words = (A.n_kv + 31) / 32 - A.prompt / 32;
    // Of the prompt two workgroups a compute unit where each has 1024 cells and more (64 tokens of 64 / 8 heads of 128 values, 32000 cells: 129 us, with one 139), else one, since every part is written and read once more (32 such tokens,
    // 8000 cells: 33 us, with two 41; 1 token, 16000 cells: 23 and 25), and 256 cells and more in each (24 tokens of 32 heads, 2047 cells: 18 us, with 128 cells 23).  Of a token's own cells four waves' worth of what is left of two
    // workgroups a compute unit; of the mask 16 words and more each, fewer for few tokens, whose words are fuller (64 / 8 heads of 128 values: 1 token of 400 cells 12 us by 2 words, 20 by 16; 4 tokens of 400 10.6 by 4, 11.2 by 8, 13.0 by 16;
    // 8 of 200 behind 1000 17 by 2, 13.0 by 8 and 13.2 by 16)
    A.prompt_parts = A.own_parts = 0;
    A.prompt_share = A.own_share = 1;
    if (A.prompt > 0) {
        const int64_t two = std::min<int64_t>(PX_PARTS - 64, target / units), most = A.prompt / std::max<int64_t>(1, two) >= 1024 ? two : target / 2 / units;
        A.prompt_share = px_share_of(A.prompt, 32, (int) std::max<int64_t>(1, std::min<int64_t>(most, (A.prompt + 255) / 256)));
        A.prompt_parts = (A.prompt + A.prompt_share - 1) / A.prompt_share;
    }
    // A single token behind a short prompt: both by the same workgroup, with nothing left to merge (32 / 4 heads of 64 values, 500 cells and 13 of its own: 8.2 us, in parts 9.9; of 250 cells 7.2 and 10.0; 64 / 8 heads of 128 values,
    // 250 cells: 9.5 and 10.9; but 500 cells 11.9 and 11.0, and 8 / 2 heads of 256 values, 500 cells: 22.6 and 15.4)
    A.together = A.n_tok == 1 && A.group <= 32 && A.prompt > 0 && A.prompt <= 512 && A.prompt * A.dim <= 32768 && A.n_kv > A.prompt && A.n_kv - A.prompt <= 256;
    if (A.together) { A.prompt_parts = 1; A.prompt_share = A.prompt; }
    else if (A.n_kv > A.prompt) {
        const int64_t left = std::max<int64_t>(4 * (target - A.prompt_parts * units), own);          // (waves of workgroups that run beside the prompt's)
        const int64_t most = std::min<int64_t>(left / own, PX_PARTS - A.prompt_parts);
        const int least = std::min(16, 2 * A.n_tok);
        A.own_share = px_share_of(words, 2, (int) std::max<int64_t>(1, std::min<int64_t>(most, (words + least - 1) / least)));
        A.own_parts = (words + A.own_share - 1) / A.own_share;
    } else if (device && A.prompt > 0) A.own_parts = 1;
    A.by_group = px_divide_by(A.group); A.by_kv = px_divide_by(A.kv); A.by_row_blocks = px_divide_by(std::max(1, A.row_blocks)); A.by_own_blocks = px_divide_by(A.own_blocks); A.by_own_parts = px_divide_by(std::max(1, A.own_parts));
    A.by_parts = px_divide_by(std::max(1, A.prompt_parts + A.own_parts)); A.by_quads = px_divide_by(A.dim / 4);
}

static int px_sizes(const char * what, int dim, int heads, int kv, int n_tok, int prompt, int n_kv) {
    if (heads < 1 || kv < 1 || heads % kv || dim < 8 || dim > 256 || dim % 8) { pi_set_error("%s: %d query heads over %d key / value heads of %d values (whole groups; 8 .. 256 values in steps of 8)", what, heads, kv, dim); return -1; }
    if ((int64_t) kv * dim > 1 << 22) { pi_set_error("%s: cells of %d x %d values", what, kv, dim); return -1; }
    if (n_tok < 0 || prompt < 0 || prompt > n_kv || n_kv > 0x7fffff00 || (int64_t) n_tok * heads > 0x3fffffff) { pi_set_error("%s: %d tokens of %d heads, %d of %d cells shared", what, n_tok, heads, prompt, n_kv); return -1; }
    return 0;
}

static size_t px_floats(const px_args & A) {
    const size_t parts = (size_t) A.prompt_parts + A.own_parts;
    return parts > 1 ? parts * A.n_tok * A.heads * (A.dim + 2) : 0;
}

extern "C" size_t pi_op_prefix_attention_scratch_floats(int head_dim, int n_head, int n_head_kv, int n_tok, int n_prompt, int n_kv) {
    if (px_sizes("pi_op_prefix_attention_scratch_floats", head_dim, n_head, n_head_kv, n_tok, n_prompt, n_kv) != 0 || n_tok == 0) return 0;
    px_args A{};
    A.dim = head_dim; A.heads = n_head; A.kv = n_head_kv; A.group = n_head / n_head_kv; A.n_tok = n_tok; A.prompt = n_prompt; A.n_kv = n_kv;
    px_plan(A, true);
    return px_floats(A);
}

template <int DP> static int px_launch(const px_args & A, hipStream_t s) {
    const int64_t own = (int64_t) A.n_tok * A.kv * A.own_blocks * A.own_parts, blocks = (int64_t) A.kv * A.prompt_parts * A.row_blocks + (own + 3) / 4;
    if (blocks > 0x1fffffff || own > 0x3fffffff) { pi_set_error("pi_op_prefix_attention: %lld workgroups", (long long) blocks); return -1; }
    const int parts = A.prompt_parts + A.own_parts, nta = std::min(A.n_tok, PI_KT_MAXNT - 1), acct = pi_account_n_kv() > 0 ? pi_account_n_kv() : A.n_kv;
    const double bytes = 4.0 * acct * A.row + 6.0 * A.n_tok * A.heads * A.dim;
    if (blocks > 0) {
        if (A.wide) PI_KT_LAUNCH(PI_KT_ATT, 0, nta, bytes, (k_prefix_attention<DP, true>), dim3((unsigned) blocks), dim3(256), 0, s, A, pi_abort_word());
        else PI_KT_LAUNCH(PI_KT_ATT, 0, nta, bytes, (k_prefix_attention<DP, false>), dim3((unsigned) blocks), dim3(256), 0, s, A, pi_abort_word());
        PI_CHECK_LAUNCH();
    }
    if (parts != 1) {
        const int at_once = 256 / (A.dim / 4);
        int groups = 0;                                      // (as a power of two)
        while (4 << groups < parts && 2 << groups <= at_once) groups++;
        const int here = at_once >> groups;
        const int64_t grid = ((int64_t) A.n_tok * A.heads + here - 1) / here;
        PI_KT_LAUNCH(PI_KT_ATT, 0, nta, 4.0 * A.n_tok * A.heads * ((double) parts * (A.dim + 2) + A.dim), k_prefix_merge, dim3((unsigned) grid), dim3(256), 0, s, A, parts, groups, here, pi_abort_word());
        PI_CHECK_LAUNCH();
    }
    return 0;
}

#define PX_BY_DIM(GO) (A.dim <= 32 ? GO(32) : A.dim <= 64 ? GO(64) : A.dim <= 96 ? GO(96) : A.dim <= 128 ? GO(128) : A.dim <= 192 ? GO(192) : GO(256))

extern "C" int pi_op_prefix_attention(const uint16_t * q16, int64_t q_stride, const uint16_t * k_cache, const uint16_t * v_cache, const uint32_t * mask, float scale, int head_dim, int n_head, int n_head_kv, int n_tok, int n_prompt,
                                      int n_kv, float * scratch, size_t scratch_floats, float * out, int64_t out_stride, float * lse, const int32_t * dyn, void * stream) {
    const char * what = "pi_op_prefix_attention";
    if (px_sizes(what, head_dim, n_head, n_head_kv, n_tok, n_prompt, n_kv) != 0) return -1;
    if (!(scale > 0.0f) || !std::isfinite(scale * 1.44269504f)) { pi_set_error("%s: scale %g (positive)", what, (double) scale); return -1; }
    if (n_tok == 0) return 0;
    if (!q16 || !out || (n_kv > 0 && (!k_cache || !v_cache)) || (!mask && n_kv > n_prompt)) { pi_set_error("%s: queries, caches, output or mask are NULL", what); return -1; }
    if (q_stride < (int64_t) n_head * head_dim || q_stride % 8 || out_stride < (int64_t) n_head * head_dim || out_stride % 4 || (((uintptr_t) q16 | (uintptr_t) k_cache | (uintptr_t) v_cache | (uintptr_t) out) & 15)) {
        pi_set_error("%s: rows of queries and outputs hold %d heads, %lld / %lld values apart (multiples of 8 / 4), all on 16 bytes", what, n_head, (long long) q_stride, (long long) out_stride);
        return -1;
    }
    px_args A{};
    A.q = q16; A.q_stride = q_stride; A.k = k_cache; A.v = v_cache; A.row = (int64_t) n_head_kv * head_dim; A.mask = mask; A.dyn = dyn; A.c = scale * 1.44269504f;
    A.dim = head_dim; A.heads = n_head; A.kv = n_head_kv; A.group = n_head / n_head_kv; A.n_tok = n_tok; A.prompt = n_prompt; A.n_kv = n_kv; A.out = out; A.out_stride = out_stride; A.lse = lse;
    px_plan(A, dyn && mask);
    const size_t need = px_floats(A);
    if (need > 0 && (!scratch || ((uintptr_t) scratch & 15) || scratch_floats < need)) { pi_set_error("%s: %zu floats of scratch, on 16 bytes, for %zu (pi_op_prefix_attention_scratch_floats)", what, scratch ? scratch_floats : 0, need); return -1; }
    A.parts_o = scratch;
    A.parts_ml = (float2 *) (scratch + (need > 0 ? (size_t) (A.prompt_parts + A.own_parts) * n_tok * n_head * head_dim : 0));
#define PX_GO(D) px_launch<D>(A, (hipStream_t) stream)
    return PX_BY_DIM(PX_GO);
#undef PX_GO
}

// ---- what cells are given ---------------------------------------------------------------------------------------------------------------------------------------------------------------
// A wave keeps the keys of 64 cells as operands and the queries of the rows go past it, 64 at a time through LDS for the four waves: a lane has 32 cells of one row of 32, adds their weights up row after row, and the lanes meet at the end.
// Bound by the clocks of the matrix cores (27 %) and the vector unit (49 %: a factor, an exponential and a sum for every score), which hardly run at once: 64 tokens of 64 / 8 heads of 128 values, 16000 cells 44 us, 17 GFLOP (rows that give nothing are looked for at every step: 1 us of it).  With the cells
// on the lanes, one sum for each and a third fewer instructions, and with three waves of it on a SIMD, the time was the same, under masks 8 % longer.  8 tokens of 32 heads, 3000 cells: 10 us, the chain from the arguments to the first keys
struct pm_args {
    const uint16_t * q; int64_t q_stride;
    const uint16_t * k; int64_t row;
    const uint32_t * mask; const float * lse; const int32_t * dyn;
    float c;
    int dim, heads, kv, group, n_tok, prompt, n_kv, cell_blocks, row_parts, row_share;
    px_div by_group, by_kv, by_blocks;
    float decay, * parts, * mass;                            // [row part][key head][cell]; null: the result is whole
};

template <int DP> __global__ void __launch_bounds__(256, DP <= 128 ? 2 : 1) k_attention_mass(const pm_args A, const int32_t * __restrict__ abort_w) {
    if (pi_aborted(abort_w, 5)) return;
    constexpr int KS = px_lds<DP>::K, N = DP / 32, CH = DP / 8, STAGE = 64 * KS;
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * STAGE > 4 * 32 * 272 ? 2 * STAGE : 4 * 32 * 272];
    __shared__ float lse[2][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, g = lane >> 5;
    const int n_kv = A.dyn ? max(0, min(A.dyn[1], A.n_kv)) : A.n_kv, prompt = min(A.dyn ? max(0, min(A.dyn[0], A.prompt)) : A.prompt, n_kv), words = (A.n_kv + 31) / 32;
    const uint32_t up = px_quotient(blockIdx.x, A.by_blocks), part = px_quotient(up, A.by_kv);
    const int cb = (int) (blockIdx.x - up * A.cell_blocks), kvh = (int) (up - part * A.kv);
    const int cells0 = cb * 256, mine = cells0 + wave * 64;
    if (cells0 >= n_kv) return;                              // (nothing of these cells is read or written: k_mass_merge stops there too)
    int r0, r1;
    px_share(A.n_tok * A.group, A.row_share, (int) part, r0, r1);
    px_u32x4 key[2][DP / 16], qr[N];
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const uint16_t * k = A.k + (int64_t) min(mine + 32 * u + n, n_kv - 1) * A.row + kvh * A.dim;
#pragma unroll
        for (int i = 0; i < DP / 16; i++) key[u][i] = px_chunk(k, 16 * i + 8 * g, A.dim);
    }
    const bool masked = cells0 + 256 > prompt, own = A.mask && n_kv > prompt;             // (without a mask nobody sees a cell behind the prompt)
    float next_lse = INFINITY;
    uint32_t ahead[2][2] = {};                                 // the mask's words of the rows on their way, lane n's row, the wave's two blocks of cells
    auto load = [&](int r) __attribute__((always_inline)) {
        if (masked && own)
#pragma unroll
            for (int v = 0; v < 2; v++) {
                const uint32_t * row = A.mask + (int64_t) px_quotient((uint32_t) min(r + 32 * v + n, r1 - 1), A.by_group) * words;
#pragma unroll
                for (int u = 0; u < 2; u++) ahead[v][u] = row[min(mine / 32 + u, words - 1)];
            }
#pragma unroll
        for (int i = 0; i < N; i++) {
            // (past the head's end the keys are zero; what is multiplied there is the head's first values)
            const int x = i * 256 + tid, d = x % CH * 8, m = min(r + x / CH, r1 - 1);
            const int t = (int) px_quotient((uint32_t) m, A.by_group);
            qr[i] = *(const px_u32x4 *) (A.q + t * A.q_stride + (int64_t) (kvh * A.group + m - t * A.group) * A.dim + (d < A.dim ? d : 0));
        }
        if (tid < 64) {
            const int m = min(r + tid, r1 - 1), t = (int) px_quotient((uint32_t) m, A.by_group);
            const float x = A.lse[(int64_t) t * A.heads + kvh * A.group + m - t * A.group];
            next_lse = r + tid >= r1 || x == -INFINITY ? INFINITY : x * 1.44269504f;      // (a row that saw nothing gives nothing)
        }
    };
    auto store = [&](int to) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < N; i++) { const int x = i * 256 + tid; *(px_u32x4 *) (lds + to * STAGE + x / CH * KS + x % CH * 16) = qr[i]; }
        if (tid < 64) lse[to][tid] = next_lse;
    };
    px_f32x16 sum[2] = { px_zero(), px_zero() };
    if (r0 < r1) { load(r0); store(0); }
    int cur = 0;
    for (int r = r0; r < r1; r += 64, cur ^= 1) {
        __syncthreads();
        const bool more = r + 64 < r1;
        const uint32_t sees[2][2] = { { ahead[0][0], ahead[0][1] }, { ahead[1][0], ahead[1][1] } };
        const float of_rows[2] = { lse[cur][n], lse[cur][32 + n] };
        if (more) load(r + 64);
        // (cells that every row sees, rows that all give something have no test: half of the vector instructions are exponentials' then)
        auto rows = [&](auto with_mask) __attribute__((always_inline)) {
#pragma unroll
            for (int v = 0; v < 2; v++) {
                if (r + 32 * v >= r1) continue;
                const uint8_t * qt = lds + cur * STAGE + (32 * v + n) * KS + 16 * g;
                const float l = of_rows[v];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int base = mine + 32 * u;
                    uint32_t bits = ~0u;
                    if constexpr (with_mask) {
                        bits = 0;
                        if (base < n_kv) {
                            if (own && base + 32 > prompt) bits = sees[v][u];
                            if (base < prompt) bits |= base + 32 > prompt ? (1u << (prompt - base)) - 1 : ~0u;
                            if (n_kv - base < 32) bits &= (1u << (n_kv - base)) - 1;
                            if (l == INFINITY) bits = 0;     // (a row that gives nothing, whatever its queries hold)
                        }
                        if (!__any(bits != 0)) continue;
                    }
                    px_f32x16 s = px_zero();
#pragma unroll
                    for (int i = 0; i < DP / 16; i++) s = px_mfma(key[u][i], *(const px_u32x4 *) (qt + 32 * i), s);
                    if constexpr (with_mask) {
                        bits >>= 4 * g;
#pragma unroll
                        for (int i = 0; i < 16; i++) if (!(bits >> (8 * (i >> 2) + (i & 3)) & 1)) s[i] = -INFINITY;
                    }
#pragma unroll
                    for (int i = 0; i < 16; i++) sum[u][i] += __builtin_amdgcn_exp2f(fmaf(s[i], A.c, -l));
                }
            }
        };
        if (masked || __any((r + n < r1 && of_rows[0] == INFINITY) || (r + 32 + n < r1 && of_rows[1] == INFINITY))) rows(std::true_type{}); else rows(std::false_type{});
        if (more) store(cur ^ 1);
    }
    // a lane has 32 cells of one row of 32: through LDS, [row of 32][cell], to one cell a lane
    __syncthreads();
    float * const at = (float *) lds + wave * (32 * 68);        // (rows 68 floats apart: sixteen bytes further round the banks)
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) *(px_f32x4 *) (at + n * 68 + 32 * u + px_cell(i, g)) = px_f32x4{ sum[u][i], sum[u][i + 1], sum[u][i + 2], sum[u][i + 3] };
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    float x[4] = { 0.0f, 0.0f, 0.0f, 0.0f };
#pragma unroll
    for (int i = 0; i < 32; i++) x[i & 3] += at[i * 68 + lane];
    const float all = (x[0] + x[1]) + (x[2] + x[3]);
    const int cell = mine + lane;
    if (cell >= n_kv) return;
    if (A.parts) A.parts[((int64_t) part * A.kv + kvh) * A.n_kv + cell] = all;
    else A.mass[cell] = A.decay == 0.0f ? all : A.decay * A.mass[cell] + all;
}

__global__ void __launch_bounds__(256) k_mass_merge(const pm_args A, int parts, const int32_t * __restrict__ abort_w) {
    if (pi_aborted(abort_w, 5)) return;
    const int n_kv = A.dyn ? max(0, min(A.dyn[1], A.n_kv)) : A.n_kv;
    const int64_t cell = (int64_t) blockIdx.x * 256 + threadIdx.x;
    if (cell >= n_kv) return;
    float x = 0.0f;
#pragma unroll 16
    for (int p = 0; p < parts; p++) x += A.parts[(int64_t) p * A.n_kv + cell];
    A.mass[cell] = A.decay == 0.0f ? x : A.decay * A.mass[cell] + x;
}

static void pm_plan(pm_args & A) {
    const int rows = A.n_tok * A.group;
    A.cell_blocks = (A.n_kv + 255) / 256;
    // as many parts of the rows as leave the fewest workgroup rounds of the chip's two per compute unit idle, at most one for every 64 rows (64 tokens of 64 / 8 heads of 128 values, 1000 cells: one part 24 us, four 11, eight 12; 4000 cells 24, 15 and 18; 16000
    // cells one or two parts 46 .. 50 us, eight 75)
    const int64_t units = (int64_t) A.cell_blocks * A.kv, slots = 2 * pi_cu_count();
    A.row_parts = 1;
    double least = 1e30;
    for (int p = 1; p <= 16 && p <= (rows + 63) / 64; p++) { const double t = (double) ((units * p + slots - 1) / slots) * (1.0 / p + 0.03); if (t < least * 0.98) { least = t; A.row_parts = p; } }
    A.row_share = px_share_of(std::max(1, rows), 64, A.row_parts);
    A.row_parts = std::max(1, (rows + A.row_share - 1) / A.row_share);
    A.by_group = px_divide_by(A.group); A.by_kv = px_divide_by(A.kv); A.by_blocks = px_divide_by(std::max(1, A.cell_blocks));
}
static size_t pm_floats(const pm_args & A) { const size_t parts = (size_t) A.kv * A.row_parts; return parts > 1 ? parts * A.n_kv : 0; }

extern "C" size_t pi_op_attention_mass_scratch_floats(int head_dim, int n_head, int n_head_kv, int n_tok, int n_prompt, int n_kv) {
    if (px_sizes("pi_op_attention_mass_scratch_floats", head_dim, n_head, n_head_kv, n_tok, n_prompt, n_kv) != 0 || n_tok == 0 || n_kv == 0) return 0;
    pm_args A{};
    A.kv = n_head_kv; A.group = n_head / n_head_kv; A.n_tok = n_tok; A.n_kv = n_kv;
    pm_plan(A);
    return pm_floats(A);
}

template <int DP> static int pm_launch(const pm_args & A, hipStream_t s) {
    const int64_t blocks = (int64_t) A.cell_blocks * A.kv * A.row_parts;
    if (blocks > 0x7fffffff) { pi_set_error("pi_op_attention_mass: %lld workgroups", (long long) blocks); return -1; }
    const int nta = std::min(A.n_tok, PI_KT_MAXNT - 1), parts = A.kv * A.row_parts;
    PI_KT_LAUNCH(PI_KT_ATT, 0, nta, 2.0 * (pi_account_n_kv() > 0 ? pi_account_n_kv() : A.n_kv) * A.row + 2.0 * A.n_tok * A.heads * A.dim, (k_attention_mass<DP>), dim3((unsigned) blocks), dim3(256), 0, s, A, pi_abort_word());
    PI_CHECK_LAUNCH();
    if (A.parts) {
        PI_KT_LAUNCH(PI_KT_ATT, 0, nta, 4.0 * A.n_kv * (parts + 2.0), k_mass_merge, dim3((unsigned) A.cell_blocks), dim3(256), 0, s, A, parts, pi_abort_word());
        PI_CHECK_LAUNCH();
    }
    return 0;
}

extern "C" int pi_op_attention_mass(const uint16_t * q16, int64_t q_stride, const uint16_t * k_cache, const uint32_t * mask, const float * lse, float scale, int head_dim, int n_head, int n_head_kv, int n_tok, int n_prompt, int n_kv,
                                    float decay, float * scratch, size_t scratch_floats, float * mass, const int32_t * dyn, void * stream) {
    const char * what = "pi_op_attention_mass";
    if (px_sizes(what, head_dim, n_head, n_head_kv, n_tok, n_prompt, n_kv) != 0) return -1;
    if (!(scale > 0.0f) || !std::isfinite(scale * 1.44269504f) || !std::isfinite(decay)) { pi_set_error("%s: scale %g (positive), decay %g", what, (double) scale, (double) decay); return -1; }
    if (n_tok == 0 || n_kv == 0) return 0;
    if (!q16 || !k_cache || !lse || !mass || (!mask && n_kv > n_prompt)) { pi_set_error("%s: queries, keys, lse, mass or mask are NULL", what); return -1; }
    if (q_stride < (int64_t) n_head * head_dim || q_stride % 8 || (((uintptr_t) q16 | (uintptr_t) k_cache) & 15)) { pi_set_error("%s: rows of queries hold %d heads, %lld values apart (a multiple of 8), queries and keys on 16 bytes", what, n_head, (long long) q_stride); return -1; }
    pm_args A{};
    A.q = q16; A.q_stride = q_stride; A.k = k_cache; A.row = (int64_t) n_head_kv * head_dim; A.mask = mask; A.lse = lse; A.dyn = dyn; A.c = scale * 1.44269504f;
    A.dim = head_dim; A.heads = n_head; A.kv = n_head_kv; A.group = n_head / n_head_kv; A.n_tok = n_tok; A.prompt = n_prompt; A.n_kv = n_kv; A.decay = decay; A.mass = mass;
    pm_plan(A);
    const size_t need = pm_floats(A);
    if (need > 0 && (!scratch || scratch_floats < need)) { pi_set_error("%s: %zu floats of scratch for %zu (pi_op_attention_mass_scratch_floats)", what, scratch ? scratch_floats : 0, need); return -1; }
    A.parts = need > 0 ? scratch : nullptr;
#define PM_GO(D) pm_launch<D>(A, (hipStream_t) stream)
    return PX_BY_DIM(PM_GO);
#undef PM_GO
}
