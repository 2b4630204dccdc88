#pragma once
// Attention of a batch of drafted trees over the cache that holds their
// sequences (ullm_hip_attn_tree, ullm_hip_attn_tree_paged).
//
// Node i of sequence b, at position p_i, sees keys t < len_b (the sequence's
// own; with a window W those with t > p_i - W) and of the keys len_b + j the
// nodes j whose bit its mask has (p_j > p_i - W):
//   out[b,i,h] = sum_t softmax_t(scale * q[b,i,h] . K[t]) V[t]
// over those, and zeros where there is none or i >= n_b.
//
// One pass over the keys with a running maximum and sum.  The rows of a kv head
// are its nodes times the G query heads that share it, row r = node r / G, head
// r % G; all of them see the same keys but for the mask, so K and V are read
// once for as many rows as a workgroup holds.
//  * S^T[16 keys x 16 rows] = K . Q^T and O^T[16 d x 16 rows] += V^T . P^T run
//    on 16x16 matrix instructions.  A lane's column is one row in both, so a
//    row's maximum, sum and rescale live in the four lanes that own its output,
//    and P^T is the S^T accumulator exponentiated: P never moves between lanes.
//    16-bit caches: 16x16x32, K by 16-byte LDS reads, V^T by the transposing
//    LDS read, P as two 16-bit values hi + lo whatever the output's type.  (P as one
//    puts outputs 1.37 times as far from 64 bits over bf16, and 1.27 over f16, as their
//    own rounding does; two take 260 us for 200 in the largest case below, where the
//    products bind, 25.3 for 24.7 and 13.1 for 12.8 in the others.)
//    f32, few rows: 16x16x4 products of f32, K and V by 16-byte reads, the four elements
//    of a read being four k-steps (K) or four d tiles (V); they run at a sixteenth of the
//    16-bit rate, which the stream of K and V about hides up to 64 rows.  f32, more rows
//    (X3): every value as the sum of three bf16 (8 bits each, exact), six products of the
//    16-bit rate (those above 2^-24 of the whole), K and V tiles split once by the waves
//    that fetched them.
//  * K and V tiles come by LDS DMA into a ring, one 32-key block a page lookup.
//  * A workgroup is WR x WK waves of 16*NR rows: the WR waves of a key group
//    share its tiles (f32 up to 32 rows: 2 WR waves, of 16 of a tile's keys each),
//    the WK key groups take tiles in turn and are added up through LDS at the end.
//  * The keys of a sequence are cut into parts, one workgroup each, so that the
//    workgroups of all sequences are alike whatever their lengths; the lengths
//    are on the device, so every workgroup works the cut out for itself
//    (find_part).  tree_merge_kernel adds the parts up.
// Measured (trace of 400 calls back to back, this kernel without the merge): 8 sequences
// of 4K-32K, 64 nodes, 32/4 heads of 128, bf16: 261 us, 215 GFLOP of products (P.V twice)
// at 822 TFLOP/s, matrix units busy in 48% of the cycles of a busy CU, and CUs busy in 71%
// of the kernel's (the second row tile of a sequence of 40 to 56 nodes is part-filled); with
// P in one piece 206, and 224 with waves in two sets half a tile apart; 24 sequences of
// 90-1500, 7 nodes, 40/8 heads, bf16: 20.9 us, 84 MB at 4.0 TB/s, the chain of a workgroup's
// start and end being 8 of them; f32, 2 sequences of 3K-8K, 48 nodes, 32/8 heads of 64:
// 39.6 us, six products of 4.4 GFLOP at 667 TFLOP/s (with f32 products 75.6); one sequence
// of 4K, 26 nodes, 12/2 heads of 128, f16: 9.9 us, of which the launch, the first loads and
// the epilogue are 8.
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>
#include "common.hpp"
#include "mfma_util.hpp"
#include "wave.hpp"

namespace ullm {

// The keys of a call: row t of sequence b is b*seq_b + t*rb bytes into the
// cache, or slot t % P of page tab[b*tab_stride + t / P] (P = 2^shift).
struct TreeKv {
    const char *k, *v;
    int64_t rb, seq_b;
    const int32_t *tab;
    int tab_stride, shift, n_pages;
};
struct TreeArgs {
    const void *q;
    const uint32_t *mask;  // words of 32 nodes; null: node i sees the nodes up to i
    const int32_t *len, *n, *pos;
    int nodes, words, max_len, window, n_head, kv_mul;
    uint32_t inv_g;  // 2^32 / kv_mul, rounded down
    float qs;   // |scale| * log2(e)
    int neg;    // scale < 0: q enters with its sign turned
    void *out;
};
// The cut of a call: slots of work along the keys (slots == batch: sequences
// are not cut), row tiles of a kv head, blocks that a part has at least, and
// the scratch for (m, l) and O of each slot, kv head, row tile and row.
struct TreePlan {
    int batch, slots, row_tiles, n_kv, least;
    float *o;
    float2 *ml;
    int2 *seq;  // first slot and parts of each sequence
};

// One sequence: keys [lo, end) in blocks of 32 from block lo / 32 on.
struct TreeSeq {
    int n, len, end, lo, blocks;
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs &a, int b) {
    TreeSeq s;
    s.n = a.n ? min(max(a.n[b], 0), a.nodes) : a.nodes;
    s.len = min(max(a.len[b], 0), a.max_len);
    s.end = min(s.len + s.n, a.max_len);
    s.lo = a.window > 0 ? max(s.len - a.window + 1, 0) : 0;
    s.blocks = s.n > 0 && s.end > s.lo ? (s.end + 31) / 32 - s.lo / 32 : 0;
    return s;
}

__device__ __forceinline__ int lane_of(int x, int l) { return __builtin_amdgcn_readlane(x, l); }

// Which sequence and part of it slot `slot` is: parts are of at most `per`
// blocks, near the least for which all sequences' parts fit the slots.  Every
// wave finds the same (any whole number of parts cuts a sequence rightly, so the
// division need not be exact); at most 256 sequences are cut.  24 sequences take
// 11000 cycles of a workgroup's start with cross-lane sums by LDS permutes and
// steps of a sixteenth, 3000 with row shifts and the estimate below.
struct TreePart {
    int b, part, parts, slot0;
    TreeSeq sq;
};
__device__ __forceinline__ TreePart find_part(const TreeArgs &a, const TreePlan &pl, int slot) {
    if (pl.batch == 1) {
        const TreeSeq q = tree_seq(a, 0);
        const int per = max((q.blocks + pl.slots - 1) / pl.slots, pl.least), parts = max((q.blocks + per - 1) / per, 1);
        return TreePart{slot < parts ? 0 : -1, slot, parts, 0, q};
    }
    const int lane = threadIdx.x & 63;
    TreeSeq sq[4];
    int total = 0;
#pragma unroll
    for (int c = 0; c < 4; c++) {
        sq[c] = TreeSeq{};
        if (c * 64 < pl.batch) {  // uniform
            if (c * 64 + lane < pl.batch) sq[c] = tree_seq(a, c * 64 + lane);
            total += lane_of(wave_scan(sq[c].blocks), 63);
        }
    }
    int per = max((total + pl.slots - 1) / pl.slots, pl.least), parts[4];
    for (;;) {
        const float inv = __builtin_amdgcn_rcpf((float)per);
        int sum = 0;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            parts[c] = 0;
            if (c * 64 < pl.batch) {
                int n = (int)((float)sq[c].blocks * inv);
                n += n * per < sq[c].blocks;
                parts[c] = c * 64 + lane < pl.batch ? max(n, 1) : 0;
                sum += lane_of(wave_scan(parts[c]), 63);
            }
        }
        if (sum <= pl.slots) break;
        // ends: with per above every sequence's blocks there are `batch` parts
        per = max(per + 1, (int)((float)per * (float)sum / (float)pl.slots));
    }
    TreePart r{-1, 0, 0, 0, {}};
    int before = 0;
#pragma unroll
    for (int c = 0; c < 4; c++) {
        if (c * 64 >= pl.batch) break;
        const int x = wave_scan(parts[c]);
        const uint64_t at = __ballot(slot >= before + x - parts[c] && slot < before + x);
        if (at) {
            const int l = __builtin_ctzll(at);
            r.b = c * 64 + l;
            r.parts = lane_of(parts[c], l);
            r.slot0 = before + lane_of(x, l) - r.parts;
            r.part = slot - r.slot0;
            r.sq = TreeSeq{lane_of(sq[c].n, l), lane_of(sq[c].len, l), lane_of(sq[c].end, l), lane_of(sq[c].lo, l),
                           lane_of(sq[c].blocks, l)};
        }
        before += lane_of(x, 63);
    }
    return r;
}

__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

// A K tile's 16-byte chunk c of row r sits in slot c ^ tree_kswz(r), a V tile's
// in c ^ tree_vswz(r) (prefill16.hip has the rates): conflict-free for the K
// reads (16 rows, one chunk) and the transposing V reads (4 rows, two chunks).
// f32 V tiles are read a contiguous row at a time and stay plain.
template <class T, int D>
__device__ __forceinline__ int tree_kswz(int r) {
    return D * T::bytes >= 256 ? r & 15 : r & 7;
}
template <class T, int D>
__device__ __forceinline__ int tree_vswz(int r) {
    if constexpr (__is_same(T, F32)) return 0;
    return D * T::bytes >= 256 ? ((r & 7) << 1) | ((r >> 3) & 1) : r & 7;
}

// Words of one f32 or two 16-bit values: the top bit of each that is an infinity
// or NaN; a value's top bit spread over it.
template <class T>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    constexpr uint32_t m = __is_same(T, F32) ? 0x7fffffffu : 0x7fff7fffu;
    constexpr uint32_t one = __is_same(T, F32) ? 0x00800000u : __is_same(T, F16) ? 0x04000400u : 0x00800080u;
    return ((w & m) + one) & ~m;
}
template <class T>
__device__ __forceinline__ uint32_t spread(uint32_t top) {
    return top | (top - (top >> (__is_same(T, F32) ? 31 : 15)));
}
// The largest, NaN if there is one: v_maximum3_f32.  (fmaxf, which passes NaN over,
// first makes each operand quiet by an instruction of its own.)
__device__ __forceinline__ float max3(float a, float b, float c) {
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

// Two workgroups share a CU where the rings of both fit it (a workgroup of eight waves
// has it to itself).
constexpr bool tree_pairs(int rb, int wr) { return rb <= 512 && wr < 8; }
// Waves that share a tile's keys, 16 each: f32 products of few rows, whose rings leave
// room for less than a wave a SIMD (8 sequences of 4K-8K, 14 rows x 256, 4 kv heads: 163
// us with one wave a tile, 101 with two).
constexpr int tree_halves(bool f32, int wr) { return f32 && wr <= 2 ? 2 : 1; }
constexpr int tree_waves(int rb, int wr, int wk) {  // of a SIMD
    return std::max((tree_pairs(rb, wr) ? 2 : 1) * wr * wk / 4, 1);
}
template <int RB, int WR, int WK, int STAGE>
constexpr int tree_stages() {
    constexpr int n = (tree_pairs(RB, WR) ? 80 : 160) * 1024 / (WK * STAGE);
    return n > 4 ? 4 : n;
}

// Two f32 as three words of bf16 pairs that add up to them: the leading 8 bits, the
// next 8, the rest (an infinity: itself and zeros).
__device__ __forceinline__ void split3(float x0, float x1, uint32_t (&w)[3]) {
    constexpr uint32_t top = 0xffff0000u, pick = 0x07060302u;  // the upper halves of two words
    const float h0 = __uint_as_float(__float_as_uint(x0) & top), h1 = __uint_as_float(__float_as_uint(x1) & top);
    const float r0 = h0 == x0 ? 0.f : x0 - h0, r1 = h1 == x1 ? 0.f : x1 - h1;
    const float m0 = __uint_as_float(__float_as_uint(r0) & top), m1 = __uint_as_float(__float_as_uint(r1) & top);
    w[0] = __builtin_amdgcn_perm(__float_as_uint(x1), __float_as_uint(x0), pick);
    w[1] = __builtin_amdgcn_perm(__float_as_uint(r1), __float_as_uint(r0), pick);
    w[2] = __builtin_amdgcn_perm(__float_as_uint(r1 - m1), __float_as_uint(r0 - m0), pick);
}

template <class T, int D, int NR, int WR, int WK, int ODT>
__global__ __launch_bounds__(64 * WR * WK * tree_halves(__is_same(T, F32), WR),
                             tree_waves(D *T::bytes, WR, WK *tree_halves(__is_same(T, F32), WR)))
void tree_kernel(TreeArgs a, TreeKv kv, TreePlan pl) {
    constexpr bool F = __is_same(T, F32);
    constexpr int KH = tree_halves(F, WR), SH = WR * KH, GR = WK * KH;  // waves of a ring, groups of waves to add up
    constexpr int EB = T::bytes, RB = D * EB, SLOTS = RB / 16, RPI = 1024 / RB;
    constexpr int KB = WR == 8 && RB <= 256 ? 64 : 32;  // keys of a tile (256 rows x 128 of bf16, P in one piece: 240 us, with 32 keys 305)
    constexpr bool X3 = F && NR * WR > 4 && D <= 128, FM = F && !X3;
    // Where four tiles fit the ring, waves that share them take two a step: half the
    // barriers (256 rows x 128 of bf16, P in one piece: 225 us, 252 with one).
    constexpr int FIT = tree_stages<RB, WR, WK, 2 * KB * RB>(), KS = !X3 && SH > 1 && FIT >= 4 ? 2 : 1;
    constexpr int TILE = KS * KB * RB, STAGE = 2 * TILE;  // a step's tiles as fetched, K and K and V
    using CT = typename std::conditional<X3, BF16, T>::type;  // operands
    constexpr int NPL = X3 ? 3 : 1, NP = F ? NPL : 2;         // pieces of K, V and Q, and of P
    constexpr int RBC = D * CT::bytes, CTILE = KB * RBC;       // a row and a tile of one piece
    constexpr int CONV = 2 * NPL * CTILE;                      // K pieces, V pieces
    constexpr int VOFF = X3 ? NPL * CTILE : TILE;              // of V behind K
    constexpr int NST = X3 ? 1 : FIT / KS;
    constexpr int GROUP = NST * STAGE + (X3 ? 2 * CONV : 0);   // LDS of a key group
    constexpr int NI = TILE / 1024 / SH;  // DMA instructions of a wave for K, and for V
    constexpr int NS = FM ? D / 16 : D / 32;  // 16-byte reads of a K row by a lane
    constexpr int NDT = D / 16;               // 16-wide d tiles of O^T
    constexpr int ROWS = 16 * NR * WR, NT = 64 * SH * WK;
    static_assert((X3 || NST >= 2) && NI >= 1 && NI * RPI <= 32, "ring and DMA shape");
    constexpr int SMO = ROWS * (D + 4) * 4, SM = GR > 1 ? GR * (SMO + ROWS * 8) : 0;
    constexpr int LDS = WK * GROUP > SM ? WK * GROUP : SM;
    static_assert(LDS + 16 <= (tree_pairs(RB, WR) ? 80 : 160) * 1024, "LDS");
    __shared__ __attribute__((aligned(1024))) char lds[LDS];
    __shared__ int unfinite;  // a V tile had infinities or NaN taken out

    const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
    const int n16 = lane & 15, kg = lane >> 4;
    const int wr = wave % WR, wk = wave / SH, grp = wave / WR;  // grp: of the waves with all rows
    const int wi = wave % SH, half = grp % KH;                 // of the ring; of a tile's keys
    // Work items (slot, kv head, row tile), the row tiles of one K/V range next
    // to each other on one XCD (workgroups are dealt to the 8 XCDs in turn).
    const int units = pl.n_kv * pl.row_tiles;
    const int item = (int)(blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    const int slot = item / units, unit = item - slot * units;
    if (slot >= pl.slots) return;
    const int kvh = unit / pl.row_tiles, rt = unit - kvh * pl.row_tiles;
    TreePart pt{slot, 0, 1, slot, {}};
    if (pl.slots > pl.batch) pt = find_part(a, pl, slot);
    else pt.sq = tree_seq(a, slot);
    const int b = uni(pt.b), part = uni(pt.part), parts = uni(pt.parts);
    if (b < 0) return;
    if (pl.slots > pl.batch && part == 0 && unit == 0 && tid == 0) pl.seq[b] = int2{pt.slot0, parts};
    const TreeSeq &sq = pt.sq;
    const int n = uni(sq.n), len = uni(sq.len), end = uni(sq.end), blocks = uni(sq.blocks);
    const int G = a.kv_mul, rows = n * G, row0 = rt * ROWS;
    auto node_of = [&](int r) {  // r / G
        const int t = (int)__umulhi((uint32_t)r, a.inv_g);  // or one less
        return t + (r - t * G >= G);
    };
    const int64_t node_ld = (int64_t)a.n_head * D;  // elements of one node's heads
    const int64_t out0 = (int64_t)b * a.nodes * node_ld + (int64_t)kvh * G * D;
    auto out_at = [&](int r) {
        const int t = node_of(r);
        return out0 + t * node_ld + (int64_t)(r - t * G) * D;
    };
    auto store4 = [&](int64_t at, const f32x4 &o) {
        if constexpr (ODT == ULLM_DT_F32) *(f32x4 *)((float *)a.out + at) = o;
        else *(u32x2 *)((uint16_t *)a.out + at) = u32x2{pack2<T>(o[0], o[1]), pack2<T>(o[2], o[3])};
    };
    if (part == 0) {  // rows of nodes that are not there
        const int r0 = max(rows, row0), r1 = min(a.nodes * G, row0 + ROWS);
        for (int i = tid; i < (r1 - r0) * (D / 4); i += NT) store4(out_at(r0 + i / (D / 4)) + i % (D / 4) * 4, f32x4{});
    }
    if (row0 >= rows) return;

    // (behind it: the first barrier of the steps, and behind that whoever sets it; X3 finds
    // them ahead of that barrier, so its waves set it after the steps)
    if (SH > 1 && tid == 0) unfinite = 0;
    // ---- this part's tiles of KB keys, dealt to the key groups in turn ----
    constexpr int BPC = KB / 32, BPT = KS * BPC;  // blocks of a tile, of a step
    const int first = uni(sq.lo) / 32, size = ((blocks + parts - 1) / parts + BPT - 1) / BPT * BPT;
    const int blk0 = first + part * size, blk1 = min(blk0 + size, first + blocks);
    const int tiles = max(blk1 - blk0 + BPT - 1, 0) / BPT;
    const int steps = (tiles + WK - 1) / WK;

    // ---- K/V DMA: instruction i of this wave writes RPI rows of the tile from
    // row (wi*NI + i)*RPI on, lane -> (row, slot) ----
    const int rb = (int)kv.rb;
    const int drow = lane / SLOTS, dslot = lane % SLOTS;
    constexpr int WROWS = KS * KB / SH;  // rows that a wave fetches, in one block
    static_assert(32 % WROWS == 0, "rows of a wave in one block");
    const int wblk = wi * WROWS / 32;         // that block of the step
    const int wrow = wi * WROWS - wblk * 32;  // and its first row there
    int kofs[NI], vofs[NI];
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const int r = wrow + i * RPI + drow;  // in the block; the swizzles go by r % 16
        kofs[i] = r * rb + ((X3 ? dslot : dslot ^ tree_kswz<T, D>(r)) * 16);
        vofs[i] = r * rb + ((X3 ? dslot : dslot ^ tree_vswz<T, D>(r)) * 16);
    }
    char *const ring = lds + wk * GROUP;
    // Pages of 128 page numbers from pg0 on, in two registers.
    int pg0 = INT_MIN, pgv[2] = {0, 0};
    auto issue = [&](int j) __attribute__((always_inline)) {  // step j's tile into stage j % NST
        const int key0 = (blk0 + (j * WK + wk) * BPT + wblk) * 32;
        const int valid = j * WK + wk < tiles ? min(end - key0, 32) : 0;
        int64_t at;
        bool ok = valid > 0;
        if (kv.tab) {
            const int pi = key0 >> kv.shift;
            if (ok && (pi < pg0 || pi >= pg0 + 128)) {
                pg0 = pi;
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const int p = pi + c * 64 + lane;
                    pgv[c] = p < kv.tab_stride ? kv.tab[(int64_t)b * kv.tab_stride + p] : -1;
                }
            }
            const int o = ok ? pi - pg0 : 0;
            const int phys = __builtin_amdgcn_readlane(o < 64 ? pgv[0] : pgv[1], o & 63);
            ok = ok && phys >= 0 && phys < kv.n_pages;
            at = (((int64_t)phys << kv.shift) + (key0 & ((1 << kv.shift) - 1))) * kv.rb;
        } else {
            at = b * kv.seq_b + (int64_t)key0 * kv.rb;
        }
        at = ok ? at + (int64_t)kvh * RB : 0;
        const int range = ok ? (valid - 1) * rb + RB : 0;  // rows from `end` on read as zeros
        const auto kr = __builtin_amdgcn_make_buffer_rsrc(uniform_ptr(kv.k + at), 0, range, kRsrcWord3);
        const auto vr = __builtin_amdgcn_make_buffer_rsrc(uniform_ptr(kv.v + at), 0, range, kRsrcWord3);
        char *st = ring + j % NST * STAGE + wi * NI * 1024;
#pragma unroll
        for (int i = 0; i < NI; i++) dma16_cached(kr, st + i * 1024, kofs[i], 0);
#pragma unroll
        for (int i = 0; i < NI; i++) dma16_cached(vr, st + TILE + i * 1024, vofs[i], 0);
    };

    // ---- this wave's rows: Q^T operands, node, position.  Their loads go out ahead
    // of the first tiles (loads return in order), and are waited for behind them. ----
    u32x4 q[NR][NPL][NS], qf[NR][X3 ? 2 * NS : 1];
    int node[NR], pos[NR];
#pragma unroll
    for (int x = 0; x < NR; x++) {
        const int r = row0 + (x * WR + wr) * 16 + n16;  // (row tiles are dealt to the waves in turn)
        const bool ok = r < rows;
        node[x] = ok ? node_of(r) : -1;
        const char *qp = (const char *)a.q + (ok ? out_at(r) : out0) * EB;
#pragma unroll
        for (int s = 0; s < (X3 ? 2 * NS : NS); s++) {
            // X3: d = 32 s + 8 kg .. +7 of every two
            const u32x4 v = *(const u32x4 *)(qp + (X3 ? (s >> 1) * 128 + kg * 32 + (s & 1) * 16 : s * 64 + kg * 16));
            if constexpr (X3) qf[x][s] = v;
            else q[x][0][s] = v;
        }
    }
    // With a window: the rows' positions, and the last one among the workgroup's.
    int most = len;
    if (a.window > 0) {
#pragma unroll
        for (int x = 0; x < NR; x++)
            pos[x] = node[x] < 0 ? 0 : a.pos ? a.pos[(int64_t)b * a.nodes + node[x]] : len + node[x];
        const int i1 = node_of(min(row0 + ROWS, rows) - 1);
        for (int i = node_of(row0) + lane; i <= i1; i += 64)
            most = max(most, a.pos ? a.pos[(int64_t)b * a.nodes + i] : len + i);
    }

#pragma unroll
    for (int j = 0; j < (SH == 1 || X3 ? NST : NST - 1); j++)
        if (j < steps) issue(j);

#pragma unroll
    for (int x = 0; x < NR; x++) {
        pos[x] = a.window > 0 ? max(pos[x], len) : 0;
        const bool ok = node[x] >= 0;
#pragma unroll
        for (int s = 0; s < NS; s++) {
            if constexpr (X3) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const u32x4 &f = qf[x][2 * s + (i >> 1)];
                    uint32_t w[3];
                    split3(__uint_as_float(f[2 * (i & 1)]), __uint_as_float(f[2 * (i & 1) + 1]), w);
#pragma unroll
                    for (int k = 0; k < 3; k++) q[x][k][s][i] = ok ? w[k] : 0;
                }
            }
        }
    }
    if (a.neg) {
        asm volatile("");  // (a branch, not a select that would wait for q here)
#pragma unroll
        for (int x = 0; x < NR; x++)
#pragma unroll
            for (int k = 0; k < NPL; k++)
#pragma unroll
                for (int s = 0; s < NS; s++) q[x][k][s] ^= FM ? 0x80000000u : 0x80008000u;
    }
    f32x4 oacc[NR][NDT];
    float m_run[NR], l_part[NR];
#pragma unroll
    for (int x = 0; x < NR; x++) {
        m_run[x] = -INFINITY, l_part[x] = 0.f;
#pragma unroll
        for (int i = 0; i < NDT; i++) oacc[x][i] = f32x4{};
    }
    // Per-lane operand addresses within a tile: of chunk 4s + kg of K, the others 64 s
    // by exclusive or (a row of pieces is 128 bytes or more), chunks 16.. of a row 256
    // bytes on; of d tile 0 of V^T, the others 32 d likewise.
    constexpr int NKA = RBC >= 256 ? 4 : 2, NVA = RBC >= 256 ? 8 : 4;
    const int hrow = half * 16, ka = (hrow + n16) * RBC + ((kg ^ tree_kswz<CT, D>(n16)) * 16), vrow = kg * 4 + (n16 >> 2);
    const int va = FM ? VOFF + (hrow + kg * 4) * RBC + n16 * 16
                      : VOFF + vrow * RBC + ((((n16 & 3) >> 1) ^ tree_vswz<CT, D>(vrow)) * 16) + 8 * (n16 & 1);
    // Blocks from `clear0` up to `clear1` hold keys that every row of the workgroup sees.
    int clear0 = 0, last = 0;
    if (a.window > 0) {
        last = uni(wave_imax(most));
        clear0 = last - a.window + 1;
    }
    const int clear1 = len;
    // Which keys of the tile of key0 row x sees, bit c of word u being key key0 +
    // 32 u + c.  The mask's words of the tile are read ahead (`words`), so that
    // they come while the tile is cleaned.
    struct MaskWords {
        uint32_t w[BPC + 1];
    };
    auto words = [&](int node, int key0) __attribute__((always_inline)) {
        MaskWords m{};
        if (!a.mask || node < 0) return m;
        const uint32_t *w = a.mask + ((int64_t)b * a.nodes + node) * a.words;
        const int w0 = max(key0 - len, 0) >> 5;
#pragma unroll
        for (int i = 0; i <= BPC; i++) m.w[i] = w0 + i < a.words ? w[w0 + i] : 0;
        return m;
    };
    auto sees = [&](int node, int pos, int lane, int key0, const MaskWords &m, uint32_t (&see)[BPC]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < BPC; u++) {
            const int k0 = key0 + 32 * u, own = len - k0, j0 = -own;  // keys of the sequence in the block; its first node
            const uint32_t mine = own >= 32 ? ~0u : own > 0 ? (1u << own) - 1 : 0u;
            const int left = end - k0;  // keys that are there
            const uint32_t there = left >= 32 ? ~0u : left > 0 ? (1u << left) - 1 : 0u;
            uint32_t t = 0;
            if (own < 32) {
                if (!a.mask) {
                    const int c = node - j0;  // bits 0..c
                    t = c >= 31 ? ~0u : c >= 0 ? (2u << c) - 1 : 0u;
                } else if (j0 < 0) {
                    t = m.w[0] << -j0;
                } else {
                    const bool next = (j0 >> 5) > max(key0 - len, 0) >> 5;  // uniform
                    const uint32_t lo = next ? m.w[BPC - 1] : m.w[0], hi = next ? m.w[BPC] : m.w[1];
                    t = (uint32_t)((((uint64_t)hi << 32) | lo) >> (j0 & 31));
                }
            }
            uint32_t s = (mine | (t & ~mine)) & there;
            if (a.window > 0) {
                const int64_t lo = (int64_t)pos - a.window + 1 - k0;  // the window's first position, from the block's
                if (lo > 0) s &= ~(mine & (lo >= 32 ? ~0u : (1u << lo) - 1));
                if (own < 32 && last - a.window >= len) {  // the window may end among the nodes
                    const int c = lane & 31, j = j0 + c;
                    int p = k0 + c;
                    if (a.pos && j >= 0 && j < n) p = max(a.pos[(int64_t)b * a.nodes + j], len);
#pragma unroll 1
                    for (int i = 0; i < 32; i++)
                        if ((int64_t)lane_of(p, i) <= (int64_t)pos - a.window) s &= ~((1u << i) & ~mine);
                }
            }
            see[u] = node < 0 ? 0 : s;
        }
    };
    // The running maximum is raised by more than 2^kLazy at a time, and a weight is held as
    // 2^kUp of what it is to it, which the row's sum carries too.  f16 ends at 2^-24: with
    // the largest weight at 2^14 or more those of 2^-28 of it keep f16's bits and its
    // smallest step is 2^-38 of it (at 1 a long tail of weights below 2^-24 was lost).  The
    // more frequent raises take 20.8 us for 19.8 (33 nodes, window 1024, 8/4 x 256).
    constexpr float kLazy = __is_same(T, F16) ? 1.f : 8.f, kUp = __is_same(T, F16) ? 14.f : 0.f;
    constexpr int KT = KB / 16 / KH;  // 16-key tiles of S^T of this wave
    auto whole = [&](int key0) { return key0 >= clear0 && key0 + KB <= clear1; };  // every row sees the tile's keys
    bool mine = false;  // this wave took infinities or NaN out of its own tiles (X3: out of what it fetched)
    // One tile, of block `blk` on, for the first NX of the wave's row tiles.  next: the
    // step whose fetch goes out under this tile's products, if there is one.
    auto tile_of = [&](auto nxc, uint32_t sb, int blk, int next) __attribute__((always_inline)) {
        constexpr int NX = decltype(nxc)::value;
        const int key0 = blk * 32;
        const bool masked = !whole(key0);
        uint32_t see[NX][BPC];
        // Infinities and NaN in V leave a tile that some row does not see all of:
        // 0 times them would not be 0.  Who does see them gets them at the end.  (All
        // waves that share the tile write the same.)
        if (__builtin_expect(masked, 0)) {
            // (copies that the compiler does not see through: what follows from them would
            // take registers in the loop)
            int nx[NX], px[NX], ln = lane;
            asm volatile("" : "+v"(ln));
            MaskWords mw[NX];
#pragma unroll
            for (int x = 0; x < NX; x++) {
                nx[x] = node[x], px[x] = pos[x];
                asm volatile("" : "+v"(nx[x]), "+v"(px[x]));
                mw[x] = words(nx[x], key0);
            }
            if constexpr (!X3) {
                uint32_t any = 0;
                constexpr int N = KB * RB / 1024, U = N < 8 ? N : 8;  // pieces, in flight
#pragma unroll 1
                for (int i = 0; i < N; i += U) {
                    const uint32_t at = sb + VOFF + i * 1024 + ln * 16;
                    u32x4 v[U];
                    static_for<0, U>([&](auto uc) { v[decltype(uc)::value] = lds_read_b128_at<decltype(uc)::value * 1024>(at); });
                    lds_wait(v);
#pragma unroll
                    for (int k = 0; k < U; k++) {
                        uint32_t bad = 0;
#pragma unroll
                        for (int e = 0; e < 4; e++) bad |= not_finite<T>(v[k][e]);
                        any |= bad;
                        if (bad) {
#pragma unroll
                            for (int e = 0; e < 4; e++) v[k][e] &= ~spread<T>(not_finite<T>(v[k][e]));
                            lds_write_b128(at + k * 1024, v[k]);
                        }
                    }
                }
                if (__any(any != 0)) {
                    if constexpr (SH > 1) unfinite = 1;
                    else mine = true;
                }
            }
#pragma unroll
            for (int x = 0; x < NX; x++) sees(nx[x], px[x], ln, key0, mw[x], see[x]);
        }
        // ---- S^T ----
        f32x4 sacc[NX][KT];
#pragma unroll
        for (int x = 0; x < NX; x++)
#pragma unroll
            for (int t = 0; t < KT; t++) sacc[x][t] = f32x4{};
        const uint32_t kaddr = sb + ka;
        constexpr int KR = NS * NPL, CH = X3 ? 6 : NS < 4 ? NS : 4, NB = KT * KR / CH;  // reads of a key tile, of a batch
        u32x4 kb[2][CH];
        auto rdk = [&](auto bc) {
            static_for<0, CH>([&](auto ic) {
                constexpr int idx = decltype(bc)::value * CH + decltype(ic)::value, t = idx / KR, s = idx % KR / NPL;
                constexpr int c = NKA == 4 ? s & 3 : s & 1, off = NKA == 4 ? (s >> 2) * 256 : 0;
                kb[decltype(bc)::value & 1][decltype(ic)::value] =
                    lds_read_b128_at<off + t * 16 * RBC + idx % NPL * CTILE>(kaddr ^ 64 * c);
            });
        };
        // V^T operands, batch by batch: CV d tiles of one 32-key block, or one key of
        // each group (f32 products); the first goes out ahead of the softmax.
        constexpr int CV = FM ? D / 64 : X3 ? 1 : 4, NBV = FM ? 4 * KT : BPC * NDT / CV;
        const uint32_t vaddr = sb + va;
        u32x4 vf[2][FM ? CV : 1];
        u32x2 vlo[2][FM ? 1 : CV * NPL], vhi[2][FM ? 1 : CV * NPL];
        auto rdv = [&](auto bc) {
            constexpr int B = decltype(bc)::value;
            if constexpr (FM)
                static_for<0, CV>([&](auto ic) {
                    constexpr int i = decltype(ic)::value;
                    vf[B & 1][i] = lds_read_b128_at<((B >> 2) * 16 + (B & 3)) * RBC + i * 256>(vaddr);
                });
            else
                static_for<0, CV * NPL>([&](auto ic) {
                    constexpr int i = decltype(ic)::value, d = B * CV % NDT + i / NPL;
                    constexpr int off = d / NVA * 256 + B * CV / NDT * 32 * RBC + i % NPL * CTILE;
                    vlo[B & 1][i] = lds_read_tr16_b64_at<off>(vaddr ^ 32 * (d % NVA));
                    vhi[B & 1][i] = lds_read_tr16_b64_at<off + 16 * RBC>(vaddr ^ 32 * (d % NVA));
                });
        };
        constexpr int VR = FM ? CV : 2 * CV * NPL;  // reads of a batch
        rdk(Int<0>{});
        static_for<0, NB>([&](auto bc) {
            constexpr int B = decltype(bc)::value;
            if constexpr (B + 1 < NB) {
                rdk(Int<B + 1>{});
                lds_wait_n<CH>();
            } else {
                rdv(Int<0>{});
                lds_wait_n<VR>();
            }
            static_for<0, CH>([&](auto ic) {
                constexpr int idx = B * CH + decltype(ic)::value, t = idx / KR, s = idx % KR / NPL, pl = idx % NPL;
                u32x4 &k = kb[B & 1][decltype(ic)::value];
                tie(k);
#pragma unroll
                for (int x = 0; x < NX; x++) {
                    if constexpr (FM) {
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            sacc[x][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[e]), __uint_as_float(q[x][0][s][e]),
                                                                              sacc[x][t], 0, 0, 0);
                    } else {
#pragma unroll
                        for (int k2 = 0; k2 + pl < NPL; k2++) sacc[x][t] = mfma16<CT>(k, q[x][k2][s], sacc[x][t]);
                    }
                }
            });
        });
        if (next < steps) issue(next);
        // ---- masks, running maximum, weights: lane = row n16, keys t*16 + kg*4 + i ----
        if (__builtin_expect(masked, 0)) {
#pragma unroll
            for (int x = 0; x < NX; x++)
#pragma unroll
                for (int u = 0; u < BPC; u++) {
                    const uint32_t s = see[x][u] >> (hrow + kg * 4);
#pragma unroll
                    for (int t = 0; t < 2 / KH; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (!(s >> (t * 16 + i) & 1)) sacc[x][2 * u + t][i] = -INFINITY;
                }
        }
        float mt[NX];
        bool up = false;
#pragma unroll
        for (int x = 0; x < NX; x++) {
            float m = -INFINITY;
#pragma unroll
            for (int t = 0; t < KT; t++) m = max3(max3(sacc[x][t][0], sacc[x][t][1], sacc[x][t][2]), sacc[x][t][3], m);
            const auto r16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(m), __float_as_uint(m), false, false);
            m = __builtin_elementwise_maximum(__uint_as_float(r16[0]), __uint_as_float(r16[1]));
            const auto r32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
            // (NaN: not above it, and the row is NaN by its sum)
            mt[x] = __builtin_elementwise_maximum(__uint_as_float(r32[0]), __uint_as_float(r32[1])) * a.qs;
            up |= mt[x] > m_run[x] + kLazy;
        }
        if (__any(up)) {
#pragma unroll
            for (int x = 0; x < NX; x++) {
                const float mn = fmaxf(m_run[x], mt[x]), mu = mn == -INFINITY ? 0.f : mn;
                const float corr = __builtin_amdgcn_exp2f(m_run[x] - mu);
                l_part[x] *= corr;
#pragma unroll
                for (int i = 0; i < NDT; i++) oacc[x][i] *= corr;
                m_run[x] = mn;
            }
        }
        u32x4 ph[NX][BPC][NP];
#pragma unroll
        for (int x = 0; x < NX; x++) {
            const float off = kUp - (m_run[x] == -INFINITY ? 0.f : m_run[x]);
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    sacc[x][t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[x][t][i], a.qs, off));
                    l_part[x] += sacc[x][t][i];
                }
            if constexpr (!FM) {
#pragma unroll
                for (int u = 0; u < BPC; u++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const f32x4 &p = sacc[x][2 * u + (i >> 1)];
                        const float p0 = p[2 * (i & 1)], p1 = p[2 * (i & 1) + 1];
                        if constexpr (NP == 3) {
                            uint32_t w[3];
                            split3(p0, p1, w);
#pragma unroll
                            for (int k = 0; k < 3; k++) ph[x][u][k][i] = w[k];
                        } else {
                            const u32x2 hl = split2<CT>(p0, p1);
                            ph[x][u][0][i] = hl[0], ph[x][u][1][i] = hl[1];
                        }
                    }
            }
        }
        // ---- O^T += V^T . P^T ----
        static_for<0, NBV>([&](auto bc) {
            constexpr int B = decltype(bc)::value;
            if constexpr (B + 1 < NBV) {
                rdv(Int<B + 1>{});
                lds_wait_n<VR>();
            } else {
                lds_wait_n<0>();
            }
            if constexpr (FM) {
#pragma unroll
                for (int i = 0; i < CV; i++) {
                    tie(vf[B & 1][i]);
#pragma unroll
                    for (int e = 0; e < 4; e++)
#pragma unroll
                        for (int x = 0; x < NX; x++)
                            oacc[x][i * 4 + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vf[B & 1][i][e]),
                                                                                      sacc[x][B >> 2][B & 3], oacc[x][i * 4 + e], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int i = 0; i < CV * NPL; i++) {
                    tie(vlo[B & 1][i]);
                    tie(vhi[B & 1][i]);
                    const u32x4 v = {vlo[B & 1][i][0], vlo[B & 1][i][1], vhi[B & 1][i][0], vhi[B & 1][i][1]};
                    constexpr int u = B * CV / NDT, d0 = B * CV % NDT;
#pragma unroll
                    for (int k = 0; k + i % NPL < NP; k++)
#pragma unroll
                        for (int x = 0; x < NX; x++) oacc[x][d0 + i / NPL] = mfma16<CT>(v, ph[x][u][k], oacc[x][d0 + i / NPL]);
                }
            }
        });
    };
    // Step j; next as above, INT_MAX: none.
    auto step = [&](int j, int next) __attribute__((always_inline)) {
        const int blk = blk0 + (j * WK + wk) * BPT;
        if (row0 + wr * 16 >= rows || blk >= blk1) {  // uniform: a wave may have no rows, or fewer than NR tiles
            if (next < steps) issue(next);
            return;
        }
        const uint32_t sb = lds_addr(ring) + (X3 ? NST * STAGE + (j & 1) * CONV : j % NST * STAGE);
#pragma unroll
        for (int s = 0; s < KS; s++) {
            if (s && blk + s * BPC >= blk1) break;
            if (NR == 1 || row0 + (WR + wr) * 16 < rows) tile_of(Int<NR>{}, sb + s * KB * RB, blk + s * BPC, s ? INT_MAX : next);
            else tile_of(Int<1>{}, sb + s * KB * RB, blk + s * BPC, s ? INT_MAX : next);
        }
    };
    // The pieces of the K and V that this wave fetched, from the f32 tile into pieces
    // (X3); the next tile is fetched as soon as they are read.
    auto convert = [&](int j) __attribute__((always_inline)) {
        const uint32_t from = lds_addr(ring) + wi * NI * 1024 + lane * 16;
        const uint32_t to = lds_addr(ring) + NST * STAGE + (j & 1) * CONV;
        const bool masked = !whole((blk0 + (j * WK + wk) * BPT) * 32);
        u32x4 x[2][NI];
        static_for<0, NI>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            x[0][i] = lds_read_b128_at<i * 1024>(from);
            x[1][i] = lds_read_b128_at<TILE + i * 1024>(from);
        });
        lds_wait_any();
        if (j + 1 < steps) issue(j + 1);
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < NI; i++)
#pragma unroll
            for (int z = 0; z < 2; z++) {
                u32x4 &v = x[z][i];
                tie(v);
                if (z == 1 && masked) {  // as above: out with V's infinities and NaN
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const uint32_t bad = spread<T>(not_finite<T>(v[e]));
                        v[e] &= ~bad;
                        any |= bad;
                    }
                }
                const int r = wblk * 32 + wrow + i * RPI + drow;  // of the tile
                uint32_t w0[3], w1[3];
                split3(__uint_as_float(v[0]), __uint_as_float(v[1]), w0);
                split3(__uint_as_float(v[2]), __uint_as_float(v[3]), w1);
                const int sw = z ? tree_vswz<CT, D>(r) : tree_kswz<CT, D>(r);
                const uint32_t at = to + z * NPL * CTILE + r * RBC + (((dslot >> 1) ^ sw) * 16) + (dslot & 1) * 8;
#pragma unroll
                for (int k = 0; k < 3; k++) lds_write_b64(at + k * CTILE, u32x2{w0[k], w1[k]});
            }
        mine |= masked && __any(any != 0);
    };

    // ---- the pipeline: one key group's wave refills a stage as soon as it has
    // read it; waves that share tiles refill behind the barrier that says that
    // all have ----
    if constexpr (X3) {
        for (int j = 0; j < steps; j++) {  // two buffers of pieces: one barrier a step
            __builtin_amdgcn_s_waitcnt(vm_wait(0));
            lds_order();
            convert(j);
            lds_wait_any();
            wg_barrier();
            step(j, INT_MAX);
        }
        if (mine) unfinite = 1;  // (then there was a step, whose barrier is behind the 0)
    } else if constexpr (SH == 1) {
        for (int j = 0; j < steps; j++) {
            if (j + NST <= steps) __builtin_amdgcn_s_waitcnt(vm_wait(std::min((NST - 1) * 2 * NI, 63)));
            else __builtin_amdgcn_s_waitcnt(vm_wait(0));
            lds_order();
            step(j, INT_MAX);
            lds_wait_any();
            if (j + NST < steps) issue(j + NST);
        }
    } else {
        for (int j = 0; j < steps; j++) {
            if (j + NST - 1 <= steps) __builtin_amdgcn_s_waitcnt(vm_wait(std::min((NST - 2) * 2 * NI, 63)));
            else __builtin_amdgcn_s_waitcnt(vm_wait(0));
            lds_wait_any();
            wg_barrier();
            step(j, j + NST - 1);
        }
    }

    // ---- infinities and NaN in V, to the rows that see their keys ----
    if constexpr (SH > 1 || WK > 1) __syncthreads();  // all tiles read, and the flag written
    if (__builtin_expect(SH > 1 ? unfinite != 0 : mine, 0)) {
#pragma unroll 1
        for (int k = 0; k < steps * BPT; k++) {
            const int t0 = blk0 + (k / BPT * WK + wk) * BPT + k % BPT / BPC * BPC, u = k % BPC;  // tile, block of it
            const int key0 = (t0 + u) * 32;
            if (t0 + u >= blk1 || whole(t0 * 32)) continue;
            uint32_t see[NR];
#pragma unroll
            for (int x = 0; x < NR; x++) {
                uint32_t s[BPC];
                sees(node[x], pos[x], lane, t0 * 32, words(node[x], t0 * 32), s);
                see[x] = u ? s[BPC - 1] : s[0];
            }
#pragma unroll 1
            for (int c = hrow; c < hrow + 32 / KH && key0 + c < end; c++) {
                int64_t at = b * kv.seq_b + (int64_t)(key0 + c) * kv.rb;
                if (kv.tab) {
                    const int pi = (key0 + c) >> kv.shift;
                    const int phys = pi < kv.tab_stride ? kv.tab[(int64_t)b * kv.tab_stride + pi] : -1;
                    if (phys < 0 || phys >= kv.n_pages) continue;
                    at = (((int64_t)phys << kv.shift) + ((key0 + c) & ((1 << kv.shift) - 1))) * kv.rb;
                }
                const char *vp = kv.v + at + (int64_t)kvh * RB + (FM ? 16 : 4) * kg * EB;
#pragma unroll
                for (int t = 0; t < NDT; t++) {
                    float v[4];
                    if constexpr (F) {
                        const f32x4 r = *(const f32x4 *)(vp + (FM ? (t >> 2) * 64 + 4 * (t & 3) : t * 16) * EB);
#pragma unroll
                        for (int e = 0; e < 4; e++) v[e] = r[e];
                    } else {
                        const u32x2 r = *(const u32x2 *)(vp + t * 16 * EB);
                        unpack2<T>(r[0], v[0], v[1]);
                        unpack2<T>(r[1], v[2], v[3]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const bool bad = not_finite<F32>(__float_as_uint(v[e]));
#pragma unroll
                        for (int x = 0; x < NR; x++) {
                            f32x4 &o = FM ? oacc[x][(t & ~3) + e] : oacc[x][t];
                            if (bad && (see[x] >> c & 1)) o[FM ? t & 3 : e] += v[e];
                        }
                    }
                }
            }
        }
    }

    // ---- results ----
    const int64_t wrow0 = ((int64_t)slot * units + unit) * ROWS;  // of the scratch
    // Element of the output (one part) or the scratch where row r of the workgroup
    // begins, < 0 for a row that is not there.
    auto row_at = [&](int r) -> int64_t { return row0 + r >= rows ? -1 : parts == 1 ? out_at(row0 + r) : (wrow0 + r) * D; };
    auto emit = [&](int64_t at, const f32x4 &o, float inv) {
        if (parts == 1) store4(at, o * inv);
        else *(f32x4 *)(pl.o + at) = o;
    };
    auto inverse = [&](float l) { return l == 0.f ? 0.f : 1.f / l; };  // (a NaN score: NaN)
#pragma unroll
    for (int x = 0; x < NR; x++) l_part[x] = rows_sum(l_part[x]);
    // Four consecutive columns from O tiles' registers: tile t (16-bit), or
    // element c % 4 of four tiles (f32 products).
    auto quad = [&](int x, int c) {
        if constexpr (FM) return f32x4{oacc[x][c & ~3][c & 3], oacc[x][(c & ~3) + 1][c & 3], oacc[x][(c & ~3) + 2][c & 3],
                                      oacc[x][(c & ~3) + 3][c & 3]};
        else return oacc[x][c];
    };
    auto qcol = [&](int c) { return FM ? (c >> 2) * 64 + 16 * kg + 4 * (c & 3) : c * 16 + kg * 4; };
    if constexpr (GR == 1) {
#pragma unroll
        for (int x = 0; x < NR; x++) {
            const int r = (x * WR + wr) * 16 + n16;
            const int64_t at = row_at(r);
            if (at < 0) continue;
            const float inv = inverse(l_part[x]);
#pragma unroll
            for (int c = 0; c < NDT; c++) emit(at + qcol(c), quad(x, c), inv);
            if (parts > 1 && kg == 0) pl.ml[wrow0 + r] = float2{m_run[x], l_part[x]};
        }
    } else {
        float *so = (float *)lds, *sml = (float *)(lds + GR * SMO);
#pragma unroll
        for (int x = 0; x < NR; x++) {
            const int r = (x * WR + wr) * 16 + n16;
#pragma unroll
            for (int c = 0; c < NDT; c++) *(f32x4 *)(so + ((int64_t)grp * ROWS + r) * (D + 4) + qcol(c)) = quad(x, c);
            if (kg == 0) *(float2 *)(sml + (grp * ROWS + r) * 2) = float2{m_run[x], l_part[x]};
        }
        __syncthreads();
        for (int r = tid; r < ROWS; r += NT) {  // the groups' weights in a row's sum
            float m = -INFINITY, l = 0.f, c[GR];
#pragma unroll
            for (int w = 0; w < GR; w++) m = fmaxf(m, sml[(w * ROWS + r) * 2]);
            const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int w = 0; w < GR; w++) {
                c[w] = __builtin_amdgcn_exp2f(sml[(w * ROWS + r) * 2] - mu);
                l += sml[(w * ROWS + r) * 2 + 1] * c[w];
            }
            const float inv = parts == 1 ? inverse(l) : 1.f;
#pragma unroll
            for (int w = 0; w < GR; w++) sml[(w * ROWS + r) * 2] = c[w] * inv;
            if (parts > 1 && row0 + r < rows) pl.ml[wrow0 + r] = float2{m, l};
        }
        __syncthreads();
        constexpr int N = ROWS * (D / 4) / NT, U = N < 4 ? N : 4;  // quads of a thread, U at a time
        static_assert(N % U == 0 && NT % (D / 4) == 0, "quads");
        const int d = tid % (D / 4) * 4;
        for (int i0 = 0; i0 < N; i0 += U) {
            f32x4 o[U];
            int64_t at[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int r = ((i0 + u) * NT + tid) / (D / 4);
                at[u] = row_at(r);
                o[u] = f32x4{};
#pragma unroll
                for (int w = 0; w < GR; w++)
                    o[u] += *(const f32x4 *)(so + ((int64_t)w * ROWS + r) * (D + 4) + d) * sml[(w * ROWS + r) * 2];
            }
#pragma unroll
            for (int u = 0; u < U; u++)
                if (at[u] >= 0) emit(at[u] + d, o[u], 1.f);
        }
    }
}

// Adds up the parts of each row of the sequences that were cut.  A row is D/4
// columns of four by 2^log_g groups of threads, each of which adds up every
// 2^log_g-th part, four parts' loads in flight; the groups meet in LDS.  Bound by
// the latency of those loads: 33 parts of 312 rows x 128 take 18.9 us with one
// group and one part at a time.
template <int D, int ODT>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a, TreePlan pl, int log_rows, int log_g) {
    constexpr int C4 = D / 4, U = 4;
    __shared__ f32x4 so[256];
    __shared__ float2 sml[256];
    const int tid = threadIdx.x, ng = 1 << log_g, c = tid % C4, g = tid / C4 & (ng - 1);
    const uint32_t row = blockIdx.x * (256 / C4 >> log_g) + (tid / C4 >> log_g);  // (node, head) of
    const int b = blockIdx.y;                                                   // this sequence
    const int2 sq = pl.seq[b];
    const int i = (int)(row / (uint32_t)a.n_head), h = (int)(row - (uint32_t)i * a.n_head);
    const int n = a.n ? min(max(a.n[b], 0), a.nodes) : a.nodes;
    if (sq.y < 2) return;  // uniform
    const bool there = i < n;
    float m = -INFINITY, l = 0.f;
    f32x4 o = {};
    if (there) {
        const int G = a.kv_mul;
        int kvh = (int)__umulhi((uint32_t)h, a.inv_g);
        kvh += h - kvh * G >= G;
        const int r = i * G + h - kvh * G, rt = r >> log_rows, units = pl.n_kv * pl.row_tiles;
        const int64_t step = (int64_t)units << log_rows;
        const int64_t at0 = sq.x * step + ((int64_t)(kvh * pl.row_tiles + rt) << log_rows) + (r & ((1 << log_rows) - 1));
        for (int p0 = g; p0 < sq.y; p0 += U * ng) {
            float2 ml[U];
            f32x4 x[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int p = p0 + u * ng;
                const int64_t at = at0 + min(p, sq.y - 1) * step;
                ml[u] = pl.ml[at];
                x[u] = *(const f32x4 *)(pl.o + at * D + c * 4);
                if (p >= sq.y) ml[u] = float2{-INFINITY, 0.f}, x[u] = f32x4{};
            }
            float mn = m;
#pragma unroll
            for (int u = 0; u < U; u++) mn = fmaxf(mn, ml[u].x);
            const float mu = mn == -INFINITY ? 0.f : mn, c0 = __builtin_amdgcn_exp2f(m - mu);
            l *= c0;
            o *= c0;
#pragma unroll
            for (int u = 0; u < U; u++) {
                const float cu = __builtin_amdgcn_exp2f(ml[u].x - mu);
                l += ml[u].y * cu;
                o += x[u] * cu;
            }
            m = mn;
        }
    }
    if (log_g) {
        so[tid] = o;
        sml[tid] = float2{m, l};
        __syncthreads();
        if (g) return;
        float mn = m;
        for (int k = 1; k < ng; k++) mn = fmaxf(mn, sml[tid + k * C4].x);
        const float mu = mn == -INFINITY ? 0.f : mn, c0 = __builtin_amdgcn_exp2f(m - mu);
        l *= c0;
        o *= c0;
        for (int k = 1; k < ng; k++) {
            const float2 ml = sml[tid + k * C4];
            const float cu = __builtin_amdgcn_exp2f(ml.x - mu);
            l += ml.y * cu;
            o += so[tid + k * C4] * cu;
        }
    }
    if (!there) return;
    f32x4 y;
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = l == 0.f ? 0.f : o[e] / l;
    const int64_t at = ((int64_t)b * a.nodes * a.n_head + row) * D + c * 4;
    if constexpr (ODT == ULLM_DT_F32) *(f32x4 *)((float *)a.out + at) = y;
    else if constexpr (ODT == ULLM_DT_F16) *(u32x2 *)((uint16_t *)a.out + at) = u32x2{pack_f16x2(y[0], y[1]), pack_f16x2(y[2], y[3])};
    else *(u32x2 *)((uint16_t *)a.out + at) = u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
}

// Waves of a workgroup (WR x WK) and 16-row tiles of a wave for `rows` rows of a
// kv head.
struct TreeShape {
    int nr, wr, wk;
    int rows() const { return 16 * nr * wr; }
};
// The widest shape for so many rows, and the next narrower one.  f32 products keep the
// matrix units busy with one row tile of a wave, so up to 64 rows are dealt to more waves.
inline TreeShape tree_shape(int dtype, int D, int rows) {
    const int rb = D * dtype_bytes(dtype);  // bytes of a key
    const int wk = rb <= 256 ? 2 : 1;       // key groups with two stages each in half a CU's LDS
    // row tiles of a wave: the registers hold no more (f32 x 128 in pieces: three times the operands)
    const int most = D == 256 || rb == 512 || (dtype == ULLM_DT_F32 && rows <= 64) ? 1 : 2;
    if (rows <= 16) return {1, 1, wk};
    if (rows <= 16 * most) return {most, 1, wk};
    int wr = 2;
    while (wr < 8 && 16 * most * wr < rows) wr *= 2;
    return {most, wr, wr <= 2 ? wk : 1};
}
inline TreeShape tree_narrower(int dtype, int D, const TreeShape &s) {
    return tree_shape(dtype, D, std::max(s.rows() / 2, 16));
}

template <class T, int D, int NR, int WR, int WK, int ODT>
static void launch_tree(const TreeArgs &a, const TreeKv &kv, const TreePlan &p, hipStream_t st) {
    const int64_t items = (int64_t)p.slots * p.n_kv * p.row_tiles;
    launch_kernel(tree_kernel<T, D, NR, WR, WK, ODT>, dim3((unsigned)((items + 7) / 8 * 8)), dim3(64 * WR * WK * tree_halves(__is_same(T, F32), WR)), 0, st,
                  a, kv, p);
    if (p.slots > p.batch) {
        constexpr int RPB = 256 / (D / 4);  // rows of a workgroup with one group each
        const int64_t rows = (int64_t)a.nodes * a.n_head;
        int log_g = 0;  // groups for four of a sequence's parts each (8 sequences of 4 parts, 16384 rows x 128: 8.8
                        // us with one group, 22.7 with eight; one sequence of 33, 312 rows: 18.9 and 5.0)
        while ((RPB >> log_g) > 1 && (4 << log_g) < p.slots / p.batch) log_g++;
        const int per = RPB >> log_g;
        launch_kernel(tree_merge_kernel<D, ODT>, dim3((unsigned)((rows + per - 1) / per), p.batch), dim3(256), 0, st, a, p,
                      __builtin_ctz(16 * NR * WR), log_g);
    }
}
template <class T, int D, int ODT>
static void launch_shape(const TreeShape &s, const TreeArgs &a, const TreeKv &kv, const TreePlan &p, hipStream_t st) {
    constexpr bool F = __is_same(T, F32);
    constexpr int rb = D * T::bytes, wide = D == 256 || rb == 512 ? 1 : 2, most = F ? 1 : wide, wk = rb <= 256 ? 2 : 1;
    if (s.wr == 8) launch_tree<T, D, wide, 8, 1, ODT>(a, kv, p, st);
    else if (s.wr == 4) {
        if (F && wide == 2 && s.nr == 2) {
            if constexpr (F && wide == 2) launch_tree<T, D, 2, 4, 1, ODT>(a, kv, p, st);
        } else {
            launch_tree<T, D, most, 4, 1, ODT>(a, kv, p, st);
        }
    } else if (s.wr == 2) launch_tree<T, D, most, 2, wk, ODT>(a, kv, p, st);
    else if (s.nr == 2) {
        if constexpr (most == 2) launch_tree<T, D, 2, 1, wk, ODT>(a, kv, p, st);
    } else {
        launch_tree<T, D, 1, 1, wk, ODT>(a, kv, p, st);
    }
}

// One call's launches (a cache type each: tree_attn_f32.hip, .._f16.hip, .._bf16.hip).
struct TreeCall {
    TreeShape shape;
    TreeArgs a;
    TreeKv kv;
    TreePlan plan;
    int head_dim;
    bool f32_out;
    hipStream_t st;
};
template <class T, int ODT>
static void launch_dims(const TreeCall &c) {
    if (c.head_dim == 64) launch_shape<T, 64, ODT>(c.shape, c.a, c.kv, c.plan, c.st);
    else if (c.head_dim == 128) launch_shape<T, 128, ODT>(c.shape, c.a, c.kv, c.plan, c.st);
    else launch_shape<T, 256, ODT>(c.shape, c.a, c.kv, c.plan, c.st);
}
void launch_tree_f32(const TreeCall &c);
void launch_tree_f16(const TreeCall &c);
void launch_tree_bf16(const TreeCall &c);

}  // namespace ullm
