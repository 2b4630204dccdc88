// The attention weight that the keys of a cache get from some rows of queries:
// ullm_hip_key_weights(_paged).
//
// The rows of a kv head are its query rows times the query heads that share it.
// A weight needs its row's denominator, which needs every score first, so a call
// goes over the keys twice: weight_rows_kernel finds each row's largest score and
// sum (log2 domain, running, split over the keys), then
//  - up to 16 rows (a decode step): it has stored its scores, 4 bytes a row and key
//    where the key itself has 2 * head_dim, and weight_sums_kernel adds them up;
//  - up to a workgroup's rows: weight_stream_kernel computes them again, the queries
//    in registers, the keys streamed;
//  - more: weight_keys_kernel, the keys in registers, the queries streamed, and
//    weight_join_kernel adds up its parts.
// Scores come from 16x16 matrix instructions; both operands are read straight from
// memory in their layout (lane l: row l % 16, 16 bytes at 64 c + 16 (l / 16)), no LDS.
// f32 queries over a 16-bit cache enter as exact pieces of its type: three of bf16, or
// two of f16 (22 bits, the row scaled by a power of two into f16's range).  An f32 cache
// takes f32 products.
#include <algorithm>
#include <climits>
#include "common.hpp"
#include "mfma_util.hpp"
#include "wave.hpp"

namespace ullm {

struct WeightArgs {
    const void *q;   // [batch][max_rows][n_head][D]
    const char *k;
    int64_t rb, seq_b;  // bytes of a cache row, from sequence to sequence
    const int32_t *tab;  // null: contiguous
    int tab_stride, shift, n_pages;
    const int32_t *len, *n_rows;
    int max_rows, max_len, window, batch, n_head, n_kv, gq;
    float qs, decay;  // scale * log2(e)
    float *w;
    int64_t w_stride;
    // how the call is cut
    int units;       // batch * n_kv
    int rows_pad;    // rows of a unit in the arrays below, a multiple of the blocks'
    int blocks;      // row blocks of a unit
    int chunk, splits;  // keys of a part of a row block, the most parts
    int row_chunk, parts;  // rows of a part of a key block, the most parts (weight_keys_kernel)
    float2 *ml;      // [units][rows_pad][splits]: largest score and sum of exp2 of a part
    float *row_qs;   // [units][rows_pad]: qs over the row's power of two
    float2 *lse;     // [units][rows_pad]: log2 of the denominator, row_qs
    float *score;    // [units][tiles][rows][16]: scores (log2 domain)
    float *part;     // [parts][units][max_len]: sums over some rows
};

// What a workgroup knows of its sequence.
struct WeightSeq {
    int len, n, rows, first;  // positions, query rows, rows of a unit, position of query row 0
    __device__ WeightSeq(const WeightArgs &a, int b) {
        len = min(max(a.len[b], 0), a.max_len);
        n = a.n_rows ? min(max(a.n_rows[b], 0), a.max_rows) : a.max_rows;
        rows = n * a.gq, first = len - n;
    }
    // Positions of rows r0 .. r1 - 1, and the keys from lo to hi that any of them sees.
    __device__ void keys(const WeightArgs &a, int r0, int r1, int &lo, int &hi) const {
        const int p0 = first + r0 / a.gq, p1 = first + (r1 - 1) / a.gq;
        hi = p1 + 1;
        lo = a.window ? max(0, p0 + 1 - a.window) : 0;
    }
};

// An operand of a row of D values of K: KC pieces of 16 bytes a lane; of a row of q NP
// times as many.
template <class TQ, class TK, int D>
struct Dot {
    static constexpr bool f32 = __is_same(TK, F32);
    static constexpr int KC = D * TK::bytes / 64;
    static constexpr int NP = f32 || __is_same(TQ, TK) ? 1 : __is_same(TK, F16) ? 2 : 3;
    static constexpr int q_regs = 4 * KC * NP;
    static constexpr int max_rt = q_regs <= 16 ? 8 : q_regs <= 32 ? 4 : q_regs <= 64 ? 2 : 1;  // row tiles of a wave
    static constexpr int kt = KC <= 4 ? 8 : KC <= 8 ? 4 : 2;  // key tiles of a wave (weight_keys_kernel)
    struct K { u32x4 x[KC]; };
    struct Q { u32x4 x[NP][KC]; };

    __device__ static void load_k(K &k, const char *row) {  // row: this lane's, its 16 bytes of each 64
#pragma unroll
        for (int c = 0; c < KC; c++) k.x[c] = *(const u32x4 *)(row + 64 * c);
    }
    // Row `row` of q (null: zeros); returns the power of two that it was divided by.
    __device__ static float load_q(Q &q, const char *row) {
        const int part = (threadIdx.x & 63) >> 4;
        if constexpr (NP == 1) {
#pragma unroll
            for (int c = 0; c < KC; c++) q.x[0][c] = row ? *(const u32x4 *)(row + 64 * c + 16 * part) : u32x4{};
            return 1.f;
        } else {
            float f = 1.f, back = 1.f;
            u32x4 raw[KC][2];
#pragma unroll
            for (int c = 0; c < KC; c++)
#pragma unroll
                for (int h = 0; h < 2; h++) raw[c][h] = row ? *(const u32x4 *)(row + 128 * c + 32 * part + 16 * h) : u32x4{};
            if constexpr (NP == 2) {
                float m = 0.f;
#pragma unroll
                for (int c = 0; c < KC; c++)
#pragma unroll
                    for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(__uint_as_float(raw[c][i >> 2][i & 3])));
                m = rows_max(m);  // the lanes of one row
                // 2^14 <= m f < 2^15 (exponents kept where f and 1 / f are normal numbers)
                const int e = min(max((int)(__float_as_uint(m) >> 23) - 127 - 14, -126), 113);
                f = __uint_as_float((uint32_t)(127 - e) << 23), back = __uint_as_float((uint32_t)(127 + e) << 23);
            }
#pragma unroll
            for (int c = 0; c < KC; c++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float x0 = __uint_as_float(raw[c][i >> 1][2 * i & 3]) * f, x1 = __uint_as_float(raw[c][i >> 1][(2 * i & 3) + 1]) * f;
#pragma unroll
                    for (int p = 0; p < NP; p++) {
                        q.x[p][c][i] = pack2<TK>(x0, x1);
                        if (p + 1 == NP) break;
                        float h0, h1;
                        unpack2<TK>(q.x[p][c][i], h0, h1);
                        x0 -= h0, x1 -= h1;
                    }
                }
            return back;
        }
    }
    // The 16x16 products of 16 keys and 16 rows: element i of lane l is key 4 (l / 16) + i of
    // row l % 16, or with ROWS row 4 (l / 16) + i of key l % 16.
    template <bool ROWS>
    __device__ static f32x4 dot(const K &k, const Q &q) {
        f32x4 s{};
#pragma unroll
        for (int p = NP - 1; p >= 0; p--)
#pragma unroll
            for (int c = 0; c < KC; c++) {
                if constexpr (f32) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float x = __uint_as_float(k.x[c][i]), y = __uint_as_float(q.x[0][c][i]);
                        s = ROWS ? __builtin_amdgcn_mfma_f32_16x16x4f32(y, x, s, 0, 0, 0)
                                 : __builtin_amdgcn_mfma_f32_16x16x4f32(x, y, s, 0, 0, 0);
                    }
                } else {
                    s = ROWS ? mfma16<TK>(q.x[p][c], k.x[c], s) : mfma16<TK>(k.x[c], q.x[p][c], s);
                }
            }
        return s;
    }
    // Row r of unit (b, g), null past the last.
    __device__ static const char *q_row(const WeightArgs &a, const WeightSeq &s, int b, int g, int r) {
        if (r >= s.rows) return nullptr;
        const int i = r / a.gq, h = r - i * a.gq;
        return (const char *)a.q + (((int64_t)b * a.max_rows + i) * a.n_head + g * a.gq + h) * D * TQ::bytes;
    }
};

// Keys of a unit, tile by tile: a wave has the pages of 2048 keys in its lanes (a page
// has 32 or more).
constexpr int kWeightKeys = 2048;
template <class P>
struct KeySource {
    const char *base;  // of the lane: its row of tile 0 of the sequence, or of the pool
    int64_t rb;
    int len, shift, n_pages, page0, pages;
    bool paged;
    __device__ KeySource(const WeightArgs &a, const WeightSeq &s, int b, int g, int k0) {
        const int lane = threadIdx.x & 63;
        paged = a.tab, rb = a.rb, len = s.len, shift = a.shift, n_pages = a.n_pages;
        base = a.k + (int64_t)g * P::KC * 64 + (lane >> 4) * 16 + (paged ? 0 : b * a.seq_b);
        page0 = k0 >> shift, pages = -1;
        if (paged && page0 + lane < a.tab_stride) pages = a.tab[(int64_t)b * a.tab_stride + page0 + lane];
    }
    // Keys t0 .. t0 + 15 (past the last: the last again).
    __device__ void load(typename P::K &k, int t0) const {
        const int t = min(t0 + (int)(threadIdx.x & 15), len - 1);
        if (!paged) {
            P::load_k(k, base + t * rb);
            return;
        }
        const int page = __builtin_amdgcn_readlane(pages, (t0 >> shift) - page0);
        if (page < 0 || page >= n_pages) {
            k = typename P::K{};
            return;
        }
        P::load_k(k, base + (((int64_t)page << shift) + (t & ((1 << shift) - 1))) * rb);
    }
};

constexpr int kWeightT = 256, kWeightW = 4;

// f(tile, its first key) over the tiles of keys k0 .. k1 - 1 that are this wave's, NB of
// them in flight.
template <class P, int NB, class F>
__device__ __forceinline__ void each_tile(const WeightArgs &a, const WeightSeq &s, int b, int g, int k0, int k1, int wave, F &&f) {
    typename P::K k[NB];
    for (int e0 = k0; e0 < k1; e0 = (e0 & -kWeightKeys) + kWeightKeys) {
        const int e1 = min(k1, (e0 & -kWeightKeys) + kWeightKeys), first = e0 + 16 * wave, last = (e1 - 1) & ~15;
        const KeySource<P> src(a, s, b, g, e0);
#pragma unroll
        for (int j = 0; j < NB; j++) src.load(k[j], min(first + 16 * kWeightW * j, last));
        for (int t0 = first; t0 < e1; t0 += 16 * kWeightW * NB)
#pragma unroll
            for (int j = 0; j < NB; j++) {
                const int t = t0 + 16 * kWeightW * j;
                if (t >= e1) break;
                f(k[j], t);
                src.load(k[j], min(t + 16 * kWeightW * NB, last));
            }
    }
}

// exp2 of a difference of scores; equal ones (also both -inf) give 1.
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float exp2_diff(float x, float m) { return x == m ? 1.f : exp2_of(x - m); }

// Largest score and sum of RT * 16 rows over a part of their keys; the four waves
// take its tiles in turn.  STORE: and the scores.  A lane's maximum is only raised where
// a score passes it by 8 (sums stay below 2^8 times their terms' count: nothing is lost).
template <class TQ, class TK, int D, int RT, bool STORE>
__global__ __launch_bounds__(kWeightT, 2) void weight_rows_kernel(WeightArgs a) {
    using P = Dot<TQ, TK, D>;
    constexpr int NB = RT * P::q_regs >= 128 ? (P::KC <= 4 ? 2 : 1) : P::KC <= 4 ? 4 : P::KC <= 8 ? 2 : 1;
    __shared__ float2 join[kWeightW][RT * 16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int unit = blockIdx.x % a.units, rest = blockIdx.x / a.units, split = rest % a.splits;
    const int r0 = (a.blocks - 1 - rest / a.splits) * RT * 16, b = unit / a.n_kv, g = unit % a.n_kv;
    const WeightSeq s(a, b);
    const int r1 = min(r0 + RT * 16, s.rows);
    if (r0 >= r1) return;
    int lo, hi;
    s.keys(a, r0, r1, lo, hi);
    const int k0 = max(lo & ~15, (lo / a.chunk + split) * a.chunk), k1 = min(hi, (lo / a.chunk + split + 1) * a.chunk);
    if (k0 >= k1) return;
    typename P::Q q[RT];
    float qs[RT], m[RT], l[RT];
    int pos[RT];
#pragma unroll
    for (int i = 0; i < RT; i++) {
        const int r = r0 + i * 16 + (lane & 15);
        qs[i] = a.qs * P::load_q(q[i], P::q_row(a, s, b, g, r));
        pos[i] = r < s.rows ? s.first + r / a.gq : -1;
        m[i] = -INFINITY, l[i] = 0.f;
    }
    // tiles that every row sees whole
    const int all_lo = a.window ? s.first + (r1 - 1) / a.gq + 1 - a.window : 0;
    const int all_hi = r1 - r0 < RT * 16 ? 0 : s.first + r0 / a.gq + 1;
    const int64_t tiles = (a.max_len + 15) >> 4;
    auto tile = [&](const typename P::K &k, int t0) {
        const bool all = t0 >= all_lo && t0 + 16 <= all_hi;
#pragma unroll
        for (int i = 0; i < RT; i++) {
            f32x4 x = P::template dot<false>(k, q[i]);
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] *= qs[i];
            if (!all) {
                const int t = t0 + 4 * (lane >> 4);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (t + j > pos[i] || (a.window && t + j <= pos[i] - a.window)) x[j] = -INFINITY;
            }
            if constexpr (STORE) {
                if ((lane & 15) < s.rows)
                    *(f32x4 *)(a.score + ((unit * tiles + (t0 >> 4)) * a.rows_pad + (lane & 15)) * 16 + 4 * (lane >> 4)) = x;
            }
            const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
            if (__any(top > m[i] + 8.f)) {
                const float up = fmaxf(m[i], top);
                l[i] *= exp2_diff(m[i], up);
                m[i] = up;
            }
            const float base = m[i] == -INFINITY ? 0.f : m[i];
            l[i] += (exp2_of(x[0] - base) + exp2_of(x[1] - base)) + (exp2_of(x[2] - base) + exp2_of(x[3] - base));
        }
    };
    each_tile<P, NB>(a, s, b, g, k0, k1, wave, tile);
#pragma unroll
    for (int i = 0; i < RT; i++) {
        const float top = rows_max(m[i]);
        const float sum = rows_sum(l[i] * exp2_diff(m[i], top));
        if (lane < 16) join[wave][i * 16 + lane] = float2{top, sum};
    }
    __syncthreads();
    if (tid < r1 - r0) {
        float top = join[0][tid].x, sum = 0.f;
        for (int w = 1; w < kWeightW; w++) top = fmaxf(top, join[w][tid].x);
        for (int w = 0; w < kWeightW; w++) sum += join[w][tid].y * exp2_diff(join[w][tid].x, top);
        a.ml[((int64_t)unit * a.rows_pad + r0 + tid) * a.splits + split] = float2{top, sum};
    }
    if (P::NP == 2 && !STORE && split == 0 && wave == 0 && lane < 16)
#pragma unroll
        for (int i = 0; i < RT; i++) a.row_qs[(int64_t)unit * a.rows_pad + r0 + i * 16 + lane] = qs[i];
}

// log2 of a row's denominator from its parts, +inf where it sees nothing (its weights
// are then 2^-inf); ROWS: rows of a block.
__device__ __forceinline__ float row_lse(const WeightArgs &a, const WeightSeq &s, int unit, int r, int block_rows) {
    if (r >= s.rows) return INFINITY;
    const int r0 = r / block_rows * block_rows;
    int lo, hi;
    s.keys(a, r0, min(r0 + block_rows, s.rows), lo, hi);
    if (hi <= lo) return INFINITY;
    const int n = (hi - 1) / a.chunk - lo / a.chunk + 1;
    const float2 *p = a.ml + ((int64_t)unit * a.rows_pad + r) * a.splits;
    float m = -INFINITY, l = 0.f;
    for (int i = 0; i < n; i++) m = fmaxf(m, p[i].x);
    for (int i = 0; i < n; i++) l += p[i].y * exp2_diff(p[i].x, m);
    return m == -INFINITY || l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

// The denominators of all rows, a thread a row.
__global__ __launch_bounds__(256) void weight_merge_kernel(WeightArgs a, int block_rows, int scaled) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= (int64_t)a.units * a.rows_pad) return;
    const int unit = (int)(at / a.rows_pad), r = (int)(at % a.rows_pad);
    const WeightSeq s(a, unit / a.n_kv);
    const float lse = row_lse(a, s, unit, r, block_rows);
    a.lse[at] = float2{lse, scaled && lse != INFINITY ? a.row_qs[at] : a.qs};
}

__device__ __forceinline__ void put_weight(const WeightArgs &a, int unit, int t, float sum) {
    float *w = a.w + (int64_t)unit * a.w_stride + t;
    *w = a.decay == 0.f ? sum : fmaf(a.decay, *w, sum);
}

// Stored scores of up to 16 rows: a thread four keys.
__global__ __launch_bounds__(kWeightT) void weight_sums_kernel(WeightArgs a) {
    __shared__ float lse[16];
    const int tid = threadIdx.x, unit = blockIdx.x % a.units, t0 = (blockIdx.x / a.units * kWeightT + tid) * 4;
    const WeightSeq s(a, unit / a.n_kv);
    if ((int)(blockIdx.x / a.units) * kWeightT * 4 >= s.len) return;
    if (tid < a.rows_pad) lse[tid] = row_lse(a, s, unit, tid, 16);
    __syncthreads();
    if (t0 >= s.len) return;
    int lo = 0, hi = 0;
    if (s.rows) s.keys(a, 0, s.rows, lo, hi);
    f32x4 sum{};
    if (t0 < hi && t0 + 3 >= (lo & ~15)) {  // (tiles that were stored)
        const float *x = a.score + (unit * (int64_t)((a.max_len + 15) >> 4) + (t0 >> 4)) * a.rows_pad * 16 + (t0 & 15);
        for (int r = 0; r < s.rows; r++) {
            const f32x4 v = *(const f32x4 *)(x + r * 16);
#pragma unroll
            for (int j = 0; j < 4; j++) sum[j] += v[j] == -INFINITY ? 0.f : exp2_of(v[j] - lse[r]);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (t0 + j < s.len) put_weight(a, unit, t0 + j, sum[j]);
}

// Weights of up to RT * 16 rows, which stay in registers, over streamed keys.
template <class TQ, class TK, int D, int RT>
__global__ __launch_bounds__(kWeightT, 2) void weight_stream_kernel(WeightArgs a) {
    using P = Dot<TQ, TK, D>;
    constexpr int NB = RT * P::q_regs >= 128 ? 1 : P::KC <= 4 ? 4 : P::KC <= 8 ? 2 : 1;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int unit = blockIdx.x % a.units, b = unit / a.n_kv, g = unit % a.n_kv;
    const WeightSeq s(a, b);
    const int k0 = blockIdx.x / a.units * a.chunk, k1 = min(s.len, k0 + a.chunk);
    if (k0 >= k1) return;
    int lo = 0, hi = 0;
    if (s.rows) s.keys(a, 0, s.rows, lo, hi);
    if (k0 >= hi || k1 <= lo) {  // no row sees these
        for (int t = k0 + tid; t < k1; t += kWeightT) put_weight(a, unit, t, 0.f);
        return;
    }
    typename P::Q q[RT];
    f32x4 lse[RT], qs[RT];
    int pos[RT];  // of the rows, four to a lane: those of the first, the others in turn
#pragma unroll
    for (int i = 0; i < RT; i++) {
        P::load_q(q[i], P::q_row(a, s, b, g, i * 16 + (lane & 15)));
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float2 x = a.lse[(int64_t)unit * a.rows_pad + i * 16 + 4 * (lane >> 4) + j];
            lse[i][j] = x.x, qs[i][j] = P::NP == 2 ? x.y : a.qs;
        }
        pos[i] = 0;
    }
    (void)pos;
    const int all_lo = a.window ? s.first + (s.rows - 1) / a.gq + 1 - a.window : 0;
    const int all_hi = s.rows < RT * 16 ? 0 : s.first + 1;
    auto tile = [&](const typename P::K &k, int t0) {
        const bool all = t0 >= all_lo && t0 + 16 <= all_hi;
        const int t = t0 + (lane & 15);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < RT; i++) {
            const f32x4 x = P::template dot<true>(k, q[i]);
            float e[4];
#pragma unroll
            for (int j = 0; j < 4; j++) e[j] = exp2_of(fmaf(x[j], qs[i][j], -lse[i][j]));
            if (!all) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int r = i * 16 + 4 * (lane >> 4) + j, p = s.first + r / a.gq;
                    if (r >= s.rows || t > p || (a.window && t <= p - a.window) || lse[i][j] == INFINITY) e[j] = 0.f;
                }
            }
            sum += (e[0] + e[1]) + (e[2] + e[3]);
        }
        sum = rows_sum(sum);
        if (lane < 16 && t < k1) put_weight(a, unit, t, sum);
    };
    each_tile<P, NB>(a, s, b, g, k0, k1, wave, tile);
}

// Sums of the weights of KT * 16 keys, which stay in registers, over row_chunk streamed
// rows; the four waves take row tiles in turn.
template <class TQ, class TK, int D>
__global__ __launch_bounds__(kWeightT, 2) void weight_keys_kernel(WeightArgs a) {
    using P = Dot<TQ, TK, D>;
    constexpr int KT = P::kt;
    __shared__ float join[kWeightW][KT * 16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int unit = blockIdx.x % a.units, rest = blockIdx.x / a.units, part = rest % a.parts, b = unit / a.n_kv, g = unit % a.n_kv;
    const int k0 = rest / a.parts * KT * 16;
    const WeightSeq s(a, b);
    const int k1 = min(k0 + KT * 16, s.len);
    if (k0 >= k1) return;
    // rows that see any of the keys
    int lo = max(part * a.row_chunk, max(0, k0 - s.first) * a.gq) & ~15, hi = min(s.rows, (part + 1) * a.row_chunk);
    if (a.window) hi = (int)min((int64_t)hi, (int64_t)max(0, k1 - 1 + a.window - s.first) * a.gq);
    float *out = a.part + ((int64_t)part * a.units + unit) * a.max_len;
    if (lo >= hi) {
        for (int t = k0 + tid; t < k1; t += kWeightT) out[t] = 0.f;
        return;
    }
    typename P::K k[KT];
    const KeySource<P> src(a, s, b, g, k0);
#pragma unroll
    for (int i = 0; i < KT; i++) src.load(k[i], min(k0 + 16 * i, (k1 - 1) & ~15));
    float sum[KT];
#pragma unroll
    for (int i = 0; i < KT; i++) sum[i] = 0.f;
    for (int r0 = lo + 16 * wave; r0 < hi; r0 += 16 * kWeightW) {
        typename P::Q q;
        P::load_q(q, P::q_row(a, s, b, g, r0 + (lane & 15)));
        float lse[4], qs[4];
        int pos[4];
        const float4 *ls = (const float4 *)(a.lse + (int64_t)unit * a.rows_pad + r0 + 4 * (lane >> 4));
        const float4 l0 = ls[0], l1 = ls[1];
        lse[0] = l0.x, lse[1] = l0.z, lse[2] = l1.x, lse[3] = l1.z;
        qs[0] = l0.y, qs[1] = l0.w, qs[2] = l1.y, qs[3] = l1.w;
        const int p0 = s.first + r0 / a.gq, p1 = s.first + (min(r0 + 16, s.rows) - 1) / a.gq;
        const bool all = r0 + 16 <= s.rows && k0 + KT * 16 - 1 <= p0 && (!a.window || k0 > p1 - a.window);
        if (!all)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int r = r0 + 4 * (lane >> 4) + j;
                pos[j] = r < s.rows && lse[j] != INFINITY ? s.first + r / a.gq : -1;
            }
#pragma unroll
        for (int i = 0; i < KT; i++) {
            const f32x4 x = P::template dot<true>(k[i], q);
            float e[4];
#pragma unroll
            for (int j = 0; j < 4; j++) e[j] = exp2_of(fmaf(x[j], qs[j], -lse[j]));
            if (!all) {
                const int t = k0 + 16 * i + (lane & 15);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (t > pos[j] || (a.window && t <= pos[j] - a.window)) e[j] = 0.f;
            }
            sum[i] += (e[0] + e[1]) + (e[2] + e[3]);
        }
    }
#pragma unroll
    for (int i = 0; i < KT; i++) {
        sum[i] = rows_sum(sum[i]);
        if (lane < 16) join[wave][i * 16 + lane] = sum[i];
    }
    __syncthreads();
    if (tid < k1 - k0) out[k0 + tid] = (join[0][tid] + join[1][tid]) + (join[2][tid] + join[3][tid]);
}

__global__ __launch_bounds__(kWeightT) void weight_join_kernel(WeightArgs a) {
    const int unit = blockIdx.x % a.units, t = blockIdx.x / a.units * kWeightT + threadIdx.x;
    const WeightSeq s(a, unit / a.n_kv);
    if (t >= s.len) return;
    float sum = 0.f;
    for (int p = 0; p < a.parts; p++) sum += a.part[((int64_t)p * a.units + unit) * a.max_len + t];
    put_weight(a, unit, t, sum);
}

// ---- how a call is cut ----
struct WeightCut {
    int rt, mode;  // row tiles of a wave; 0: scores stored, 1: rows in registers, 2: keys in registers
    int rows_pad, blocks, chunk, splits, row_chunk, parts;
    size_t ml, qs, lse, score, part, bytes;  // offsets
};
static int weight_max_rt(int q_dtype, int dtype, int D) {
    const int kc = D * dtype_bytes(dtype) / 64, np = q_dtype == dtype ? 1 : dtype == ULLM_DT_F16 ? 2 : 3, regs = 4 * kc * np;
    return regs <= 16 ? 8 : regs <= 32 ? 4 : regs <= 64 ? 2 : 1;
}
constexpr int64_t kWeightWgs = 1024;  // workgroups aimed at: two to four rounds of the card
static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
static WeightCut weight_cut(int q_dtype, int dtype, int64_t batch, int max_rows, int max_len, int window, int n_head,
                            int64_t n_kv, int D) {
    WeightCut c{};
    const int64_t rows = (int64_t)max_rows * (n_head / n_kv), units = batch * n_kv;
    const int top = weight_max_rt(q_dtype, dtype, D);
    c.rt = 1;
    while (c.rt < top && c.rt * 16 < rows) c.rt *= 2;
    c.blocks = (int)((rows + c.rt * 16 - 1) / (c.rt * 16));
    c.mode = rows <= 16 ? 0 : c.blocks == 1 ? 1 : 2;
    c.rows_pad = c.mode == 0 ? (int)rows : c.blocks * c.rt * 16;
    // parts of a row block's keys, whole tiles for every wave
    const int64_t keys = window > 0 && window < max_len ? std::min<int64_t>(max_len, (int64_t)window + max_rows) : max_len;
    const int64_t want = (keys * units * c.blocks + kWeightWgs - 1) / kWeightWgs;
    c.chunk = (int)std::max<int64_t>(std::min<int64_t>((want + 63) / 64, (max_len + 63) / 64) * 64, 128);
    c.splits = (int)((keys + c.chunk - 1) / c.chunk + (window > 0 ? 1 : 0));
    c.parts = (int)std::min<int64_t>(16, (rows + 255) / 256);
    c.row_chunk = (int)(((rows + c.parts - 1) / std::max(c.parts, 1) + 63) / 64 * 64);
    size_t at = 0;
    const size_t entries = (size_t)units * c.rows_pad;
    c.ml = at, at += up256(entries * c.splits * sizeof(float2));
    c.qs = at, at += up256(entries * sizeof(float));
    c.lse = at, at += c.mode ? up256(entries * sizeof(float2)) : 0;
    c.score = at, at += c.mode == 0 ? up256((size_t)units * ((max_len + 15) / 16) * c.rows_pad * 16 * sizeof(float)) : 0;
    c.part = at, at += c.mode == 2 ? up256((size_t)c.parts * units * max_len * sizeof(float)) : 0;
    c.bytes = at;
    return c;
}

template <class TQ, class TK, int D, int RT>
static void launch_rows(const WeightArgs &a, const WeightCut &c, hipStream_t st) {
    using P = Dot<TQ, TK, D>;
    const dim3 wg(kWeightT);
    const unsigned units = a.units;
    if (c.mode == 0) {
        if constexpr (RT == 1) {
            launch_kernel(weight_rows_kernel<TQ, TK, D, 1, true>, dim3(units * c.splits), wg, 0, st, a);
            launch_kernel(weight_sums_kernel, dim3(units * ((a.max_len + 4 * kWeightT - 1) / (4 * kWeightT))), wg, 0, st, a);
        }
        return;
    }
    launch_kernel(weight_rows_kernel<TQ, TK, D, RT, false>, dim3(units * c.splits * c.blocks), wg, 0, st, a);
    launch_kernel(weight_merge_kernel, dim3(((size_t)units * c.rows_pad + 255) / 256), dim3(256), 0, st, a, RT * 16, (int)(P::NP == 2));
    if (c.mode == 1) {
        launch_kernel(weight_stream_kernel<TQ, TK, D, RT>, dim3(units * ((a.max_len + a.chunk - 1) / a.chunk)), wg, 0, st, a);
        return;
    }
    constexpr int keys = P::kt * 16;
    launch_kernel(weight_keys_kernel<TQ, TK, D>, dim3(units * a.parts * ((a.max_len + keys - 1) / keys)), wg, 0, st, a);
    launch_kernel(weight_join_kernel, dim3(units * ((a.max_len + kWeightT - 1) / kWeightT)), wg, 0, st, a);
}
template <class TQ, class TK, int D>
static void launch_weights(const WeightArgs &a, const WeightCut &c, hipStream_t st) {
    constexpr int top = Dot<TQ, TK, D>::max_rt;
    if (c.rt == 1) launch_rows<TQ, TK, D, 1>(a, c, st);
    if constexpr (top >= 2) if (c.rt == 2) launch_rows<TQ, TK, D, 2>(a, c, st);
    if constexpr (top >= 4) if (c.rt == 4) launch_rows<TQ, TK, D, 4>(a, c, st);
    if constexpr (top >= 8) if (c.rt == 8) launch_rows<TQ, TK, D, 8>(a, c, st);
}
template <class TQ, class TK>
static void launch_weights(const WeightArgs &a, const WeightCut &c, int D, hipStream_t st) {
    if (D == 64) launch_weights<TQ, TK, 64>(a, c, st);
    else if (D == 128) launch_weights<TQ, TK, 128>(a, c, st);
    else launch_weights<TQ, TK, 256>(a, c, st);
}

static int key_weights(const char *fn, WeightArgs a, int q_dtype, int dtype, int64_t kv_stride, int head_dim,
                       float scale, void *ws, size_t ws_bytes, void *stream) {
    if (!dtype_ok(dtype) || (q_dtype != ULLM_DT_F32 && q_dtype != dtype))
        return set_error(ULLM_HIP_E_UNSUPPORTED, "%s: q of dtype %d over a cache of dtype %d", fn, q_dtype, dtype);
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return set_error(ULLM_HIP_E_UNSUPPORTED, "%s: head_dim %d not in {64,128,256}", fn, head_dim);
    if (a.batch < 0 || a.batch > 65535 || a.max_rows < 0 || a.max_len < 0 || a.window < 0)
        return set_error(ULLM_HIP_E_INVALID, "%s: batch not in 0..65535, or max_rows, max_len or window < 0", fn);
    if (a.n_head < 1 || a.n_kv < 1 || a.n_head % a.n_kv || a.n_head > 65535)
        return set_error(ULLM_HIP_E_INVALID, "%s: bad heads", fn);
    if (a.max_len > 1 << 30) return set_error(ULLM_HIP_E_INVALID, "%s: max_len %d > 2^30", fn, a.max_len);
    if (a.window >= a.max_len) a.window = 0;  // (what every row sees)
    if ((int64_t)a.max_rows * a.n_head > 1 << 23) return set_error(ULLM_HIP_E_INVALID, "%s: too many rows", fn);
    if (kv_stride < (int64_t)a.n_kv * head_dim || a.w_stride < a.max_len)
        return set_error(ULLM_HIP_E_INVALID, "%s: kv_stride or weights_stride too small", fn);
    if (a.batch == 0 || a.max_len == 0) return ULLM_HIP_OK;
    if ((!a.q && a.max_rows) || !a.k || !a.len || !a.w) return set_error(ULLM_HIP_E_INVALID, "%s: null tensor pointer", fn);
    const int eb = dtype_bytes(dtype);
    if (((uintptr_t)a.q | (uintptr_t)a.k) & 15 || kv_stride * eb % 16 || a.seq_b % 16)
        return set_error(ULLM_HIP_E_INVALID, "%s: tensors and row strides must be 16-byte aligned", fn);
    const int rows = std::max(a.max_rows, 1);  // (none: the weights fade, as n_rows of 0 does)
    const WeightCut c = weight_cut(q_dtype, dtype, a.batch, rows, a.max_len, a.window, a.n_head, a.n_kv, head_dim);
    const int64_t units = (int64_t)a.batch * a.n_kv;
    // (a grid has less than 2^32 threads)
    if (units * c.splits * c.blocks >= 1 << 24 || units * c.rows_pad > INT_MAX || units * ((a.max_len + 31) / 32) * c.parts >= 1 << 24)
        return set_error(ULLM_HIP_E_INVALID, "%s: too many rows or keys", fn);
    if (!ws || ws_bytes < c.bytes || (uintptr_t)ws & 255)
        return set_error(ULLM_HIP_E_WORKSPACE, "%s: workspace of %zu bytes, 256-byte aligned, needed", fn, c.bytes);
    a.gq = a.n_head / a.n_kv;
    a.qs = scale * kLog2e;
    a.rb = kv_stride * eb;
    a.units = (int)units, a.rows_pad = c.rows_pad, a.blocks = c.blocks, a.chunk = c.chunk, a.splits = c.splits;
    a.row_chunk = c.row_chunk, a.parts = c.parts;
    char *const at = (char *)ws;
    a.ml = (float2 *)(at + c.ml), a.row_qs = (float *)(at + c.qs), a.lse = (float2 *)(at + c.lse);
    a.score = (float *)(at + c.score), a.part = (float *)(at + c.part);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == ULLM_DT_F32) launch_weights<F32, F32>(a, c, head_dim, st);
    else if (dtype == ULLM_DT_F16) q_dtype == dtype ? launch_weights<F16, F16>(a, c, head_dim, st) : launch_weights<F32, F16>(a, c, head_dim, st);
    else q_dtype == dtype ? launch_weights<BF16, BF16>(a, c, head_dim, st) : launch_weights<F32, BF16>(a, c, head_dim, st);
    return check_hip(hipGetLastError(), "key_weights launch");
}

}  // namespace ullm

using namespace ullm;

extern "C" int ullm_hip_key_weights(const void *q, int q_dtype, const void *k_cache, int kv_dtype, int64_t kv_stride,
                                    int64_t seq_stride, const int32_t *seq_lens, const int32_t *n_rows, int max_rows,
                                    int max_len, int window, int batch, int n_head, int n_kv_head, int head_dim,
                                    float scale, float decay, float *weights, int64_t weights_stride, void *workspace,
                                    size_t workspace_bytes, void *stream) {
    if (seq_stride < 0) return set_error(ULLM_HIP_E_INVALID, "key_weights: seq_stride < 0");
    const WeightArgs a{q, (const char *)k_cache, 0, batch > 1 && dtype_ok(kv_dtype) ? seq_stride * dtype_bytes(kv_dtype) : 0,
                       nullptr, 0, 0, 0, seq_lens, n_rows, max_rows, max_len, window, batch, n_head, n_kv_head, 0, 0.f,
                       decay, weights, weights_stride};
    return key_weights("key_weights", a, q_dtype, kv_dtype, kv_stride, head_dim, scale, workspace, workspace_bytes, stream);
}

extern "C" int ullm_hip_key_weights_paged(const void *q, int q_dtype, const void *k_pages, int kv_dtype,
                                          int64_t kv_stride, int page_size, int n_pages, const int32_t *block_table,
                                          int table_stride, const int32_t *seq_lens, const int32_t *n_rows,
                                          int max_rows, int max_len, int window, int batch, int n_head, int n_kv_head,
                                          int head_dim, float scale, float decay, float *weights,
                                          int64_t weights_stride, void *workspace, size_t workspace_bytes,
                                          void *stream) {
    if (page_size < 32 || (page_size & (page_size - 1)))
        return set_error(ULLM_HIP_E_INVALID, "key_weights_paged: page_size %d must be a power of two >= 32", page_size);
    if (n_pages < 1 || table_stride < 1 || (int64_t)table_stride * page_size < max_len)
        return set_error(ULLM_HIP_E_INVALID, "key_weights_paged: n_pages %d, table of %d pages for max_len %d", n_pages,
                         table_stride, max_len);
    if (batch > 0 && max_len > 0 && !block_table)
        return set_error(ULLM_HIP_E_INVALID, "key_weights_paged: null tensor pointer");
    const WeightArgs a{q, (const char *)k_pages, 0, 0, block_table, table_stride, __builtin_ctz(page_size), n_pages,
                       seq_lens, n_rows, max_rows, max_len, window, batch, n_head, n_kv_head, 0, 0.f, decay, weights,
                       weights_stride};
    return key_weights("key_weights_paged", a, q_dtype, kv_dtype, kv_stride, head_dim, scale, workspace,
                       workspace_bytes, stream);
}

extern "C" size_t ullm_hip_key_weights_workspace_bytes(int kv_dtype, int batch, int max_rows, int max_len, int window,
                                                       int n_head, int n_kv_head, int head_dim) {
    if (!dtype_ok(kv_dtype) || (head_dim != 64 && head_dim != 128 && head_dim != 256) || batch < 1 || max_rows < 1 ||
        max_len < 1 || max_len > 1 << 30 || window < 0 || n_head < 1 || n_kv_head < 1 || n_head % n_kv_head || n_head > 65535 ||
        (int64_t)max_rows * n_head > 1 << 23)
        return 0;
    // For every call with fewer sequences, rows and positions too: parts of row blocks are at most
    // kWeightWgs and three more a block; the scores are those of up to 16 rows.
    const int gq = n_head / n_kv_head;
    const int64_t rows = (int64_t)max_rows * gq, units = (int64_t)batch * n_kv_head;
    size_t most = 0;
    for (int q_dtype : {(int)ULLM_DT_F32, kv_dtype}) {
        const int block = 16 * weight_max_rt(q_dtype, kv_dtype, head_dim);
        const int64_t blocks = (rows + block - 1) / block;
        size_t n = up256((kWeightWgs + 3 * units * blocks) * block * sizeof(float2)) + 2 * up256(units * blocks * block * sizeof(float2));
        n += std::max((size_t)(gq <= 16 ? up256((size_t)units * ((max_len + 15) / 16) * std::min<int64_t>(rows, 16) * 16 * sizeof(float)) : 0),
                      up256((size_t)std::min<int64_t>(16, (rows + 255) / 256) * units * max_len * sizeof(float)));
        most = std::max(most, n);
    }
    return most;
}
