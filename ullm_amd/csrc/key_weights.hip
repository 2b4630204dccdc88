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
// Scores come from 16x16 matrix instructions.  What is streamed comes by LDS DMA, whole
// rows to consecutive lanes, into a ring of the wave's own (no barriers), and is read
// from there in the operands' layout (lane l: row l % 16, 16 bytes at 64 c + 16 (l / 16)),
// the 16-byte columns of a row exchanged by its number so that no two lanes meet in a
// bank.  Read straight from memory in that layout, a lane's neighbours all lie in other
// rows, 64 lines a load: the last 32 rows of a 32K prompt took 77 us so, 50 with the keys
// and 38 with the queries through LDS.
// f32 queries over a 16-bit cache enter in pieces of its type: three of bf16, which hold
// all 24 bits, or two of f16, the row scaled by a power of two into f16's range.  These hold 22
// bits, off by at most 2^-23 of a value or 2^-39 of the row's largest, well inside the
// bound of a score's sum of head_dim products in 32 bits; a third piece would be half as
// many products again.  An f32 cache takes f32 products.
//
// Measured (us, 32/8 or 32/4 heads x 128, bf16): one row over 8 sequences of 4K-32K (154 MB of
// keys) 50-53: 41 to 44 in the rows (33 with their loads alone, where reads of as many bytes
// take 27; 34 with the arithmetic and no scores stored; the rest are the 19 MB of scores, written
// beside the loads and counted with them) and 9 in the sums; the last
// 32 rows of 32K 37.7: 19.8 and 17.1 over 64 MB of keys each, 4.8 in the merge; all 2048
// rows of a prompt 66 to 69: 31 and 41, vector instructions (an exponential counts four) for
// about 40 of it, a workgroup's start, 3 to 4 us, for most of the rest.  In weight_keys_kernel
// a step of 16 rows and 64 keys has 47 of the formula, 16 of them exponentials, and 36 that
// find the places of the next query rows, 8 of them whole products at an exponential's
// rate: two fifths of the step.
#include <algorithm>
#include <climits>
#include <cmath>
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
    uint32_t gq_mul;  // r / gq of a whole number r >= 0: r * gq_mul >> (32 + gq_shift), or r >> gq_shift where it is 0
    int gq_shift;
    float qs, decay;  // scale * log2(e)
    float *w;
    int64_t w_stride;
    // how the call is cut
    int units;       // batch * n_kv
    int rows_pad;    // rows of a unit in the arrays below, a multiple of the blocks'
    int blocks;      // row blocks of a unit
    int chunk, splits;  // keys of a part of a row block, the most parts
    int direct;         // one part a row block: its denominators are the rows'
    int spread;         // or: parts that all sequences have together, cut by their lengths (see weight_spread)
    int64_t tiles;  // of the scores of a unit
    int row_chunk, parts;  // rows of a part of a key block, the most parts (weight_keys_kernel)
    float2 *ml;      // [parts][rows of a block]: largest score and sum of exp2 of a part (see weight_part)
    float *row_qs;   // [units][rows_pad]: qs over the row's power of two
    float2 *lse;     // [units][rows_pad]: log2 of the denominator, row_qs
    float *score;    // [units][tiles][rows][16]: scores (log2 domain)
    float *part;     // [parts][units][max_len]: sums over some rows
};

__device__ __forceinline__ int query_row(const WeightArgs &a, int r) {
    return (a.gq_mul ? __umulhi(r, a.gq_mul) : r) >> a.gq_shift;
}

// What a workgroup knows of its sequence.
struct WeightSeq {
    int len, n, rows, first;  // positions, query rows, rows of a unit, position of query row 0
    __device__ __forceinline__ WeightSeq(const WeightArgs &a, int b) {
        len = min(max(a.len[b], 0), a.max_len);
        n = a.n_rows ? min(max(a.n_rows[b], 0), a.max_rows) : a.max_rows;
        rows = n * a.gq, first = len - n;
    }
    // Positions of rows r0 .. r1 - 1, and the keys from lo to hi that any of them sees.
    __device__ __forceinline__ void keys(const WeightArgs &a, int r0, int r1, int &lo, int &hi) const {
        const int p0 = first + query_row(a, r0), p1 = first + query_row(a, r1 - 1);
        hi = p1 + 1;
        lo = a.window ? max(0, p0 + 1 - a.window) : 0;
    }
};

// 16 rows of RB bytes in LDS: chunk (16 bytes) c of row r lies at r RB + 16 (c ^ swz(r)).
template <int RB>
struct Tile {
    static constexpr int C = RB / 16, N = RB / 64, bytes = 16 * RB;  // chunks of a row, DMA instructions of a tile
    __device__ __forceinline__ static int swz(int row) { return C == 8 ? (row >> 1) & 7 : row & 15; }
    // What lane l fetches in instruction d: its row, and its bytes in it.
    __device__ __forceinline__ static int row(int d) { return (d * 64 + (int)(threadIdx.x & 63)) / C; }
    __device__ __forceinline__ static int col(int d) { return (((int)(threadIdx.x & 63) % C) ^ swz(row(d))) * 16; }
    // Where lane l reads chunk c of row l % 16.
    __device__ __forceinline__ static uint32_t at(int c) {
        const int r = threadIdx.x & 15;
        return r * RB + ((c ^ swz(r)) * 16);
    }
};
// Waits until at most N vector-memory operations of this wave are outstanding.
template <int N>
__device__ __forceinline__ void vm_wait_n() {
    static_assert(N >= 0 && N < 64, "vmcnt");
    asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}

// An operand of a row of D values of K: KC pieces of 16 bytes a lane; of a row of q NP
// times as many.
template <class TQ, class TK, int D>
struct Dot {
    static constexpr bool f32 = __is_same(TK, F32);
    static constexpr int KC = D * TK::bytes / 64;
    static constexpr int NP = f32 || __is_same(TQ, TK) ? 1 : __is_same(TK, F16) ? 2 : 3;
    static constexpr int q_regs = 4 * KC * NP, q_bytes = D * TQ::bytes;
    // most row tiles of a wave where the rows stay in registers
    static constexpr int rt = q_regs <= 16 ? 4 : q_regs <= 48 ? 2 : 1;
    // weight_keys_kernel: key tiles of a wave
    static constexpr int kt = KC <= 2 ? 8 : KC <= 4 ? 4 : NP > 1 || KC > 8 ? 2 : 4;
    using KTile = Tile<D * TK::bytes>;
    using QTile = Tile<D * TQ::bytes>;
    static constexpr int H = KC <= 4 ? 2 : 1;  // key tiles of a step where the keys are streamed
    static constexpr int step_bytes = H * KTile::bytes;
    static constexpr int waves = step_bytes > 8192 ? 1 : 2, keys_waves = QTile::bytes > 8192 ? 1 : 2;  // of a SIMD, by the rings
    struct K { u32x4 x[KC]; };
    struct Q { u32x4 x[NP][KC]; };
    struct Raw { u32x4 x[QTile::N]; };  // chunks of a row of q: of K's type 4 c + l / 16, f32 8 (c / 2) + 2 (l / 16) + c % 2
    __device__ __forceinline__ static int raw_chunk(int c) {
        const int part = (threadIdx.x & 63) >> 4;
        return NP == 1 ? 4 * c + part : 8 * (c >> 1) + 2 * part + (c & 1);
    }
    // The operand of a row of q, of other sign if `neg`; returns the power of two that it was
    // divided by.
    __device__ __forceinline__ static float make_q(Q &q, const Raw &raw, bool neg) {
        if constexpr (NP == 1) {
#pragma unroll
            for (int c = 0; c < KC; c++) q.x[0][c] = raw.x[c];
            if (neg)
#pragma unroll
                for (int c = 0; c < KC; c++) q.x[0][c] ^= f32 ? 0x80000000u : 0x80008000u;
            return 1.f;
        } else {
            float f = 1.f, back = 1.f;
            if constexpr (NP == 2) {
                float m = 0.f;
#pragma unroll
                for (int c = 0; c < 2 * KC; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++) m = fmaxf(m, fabsf(__uint_as_float(raw.x[c][i])));
                m = rows_max(m);  // the lanes of one row
                // 2^14 <= m f < 2^15, or less where m is below 2^-46
                const int e = min(max((int)(__float_as_uint(m) >> 23) - 127 - 14, -60), 113);
                f = __uint_as_float((uint32_t)(127 - e) << 23), back = __uint_as_float((uint32_t)(127 + e) << 23);
            }
            if (neg) f = -f;
#pragma unroll
            for (int c = 0; c < KC; c++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const u32x4 &r = raw.x[2 * c + (i >> 1)];
                    float x0 = __uint_as_float(r[2 * i & 3]) * f, x1 = __uint_as_float(r[(2 * i & 3) + 1]) * f;
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
    // The 16x16 products of NK key tiles and NQ row tiles, x[i][h] of rows i and keys h: element
    // j of lane l is key 4 (l / 16) + j of row l % 16, or with ROWS row 4 (l / 16) + j of key
    // l % 16.  Tiles in turn (a tile's next product waits for its last one).
    template <bool ROWS, int NQ, int NK>
    __device__ __forceinline__ static void dots(f32x4 (&x)[NQ][NK], const K *k, const Q *q) {
#pragma unroll
        for (int i = 0; i < NQ; i++)
#pragma unroll
            for (int h = 0; h < NK; h++) x[i][h] = f32x4{};
#pragma unroll
        for (int p = NP - 1; p >= 0; p--)
#pragma unroll
            for (int c = 0; c < KC; c++)
#pragma unroll
                for (int e = 0; e < (f32 ? 4 : 1); e++)
#pragma unroll
                    for (int i = 0; i < NQ; i++)
#pragma unroll
                        for (int h = 0; h < NK; h++) {
                            f32x4 &s = x[i][h];
                            if constexpr (f32) {
                                const float a = __uint_as_float(k[h].x[c][e]), b = __uint_as_float(q[i].x[0][c][e]);
                                s = ROWS ? __builtin_amdgcn_mfma_f32_16x16x4f32(b, a, s, 0, 0, 0)
                                         : __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, s, 0, 0, 0);
                            } else {
                                s = ROWS ? mfma16<TK>(q[i].x[p][c], k[h].x[c], s) : mfma16<TK>(k[h].x[c], q[i].x[p][c], s);
                            }
                        }
    }
};

// Keys of a unit: a wave has the pages of 2048 keys in its lanes (a page has 32 or more).
constexpr int kWeightKeys = 2048;
template <class P>
struct KeySource {
    const char *base;  // of the kv head's part of row 0 of the sequence, or of the pool
    int64_t rb;
    int len, shift, n_pages, page0, pages;
    bool paged;
    __device__ __forceinline__ KeySource(const WeightArgs &a, const WeightSeq &s, int b, int g, int k0) {
        const int lane = threadIdx.x & 63;
        paged = a.tab, rb = a.rb, len = s.len, shift = a.shift, n_pages = a.n_pages;
        base = a.k + (int64_t)g * P::KC * 64 + (paged ? 0 : b * a.seq_b);
        page0 = k0 >> shift, pages = -1;
        if (paged && page0 + lane < a.tab_stride) pages = a.tab[(int64_t)b * a.tab_stride + page0 + lane];
    }
    // Keys t0 .. t0 + n - 1 (in one page); those past the last, and those of pages outside the
    // pool, read as zeros.
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows(int t0, int n) const {
        int64_t row = t0;
        int bytes = t0 < len ? (min(n, len - t0) - 1) * (int)rb + P::KC * 64 : 0;
        if (paged) {
            const int page = __builtin_amdgcn_readlane(pages, (t0 >> shift) - page0);
            const bool there = (unsigned)page < (unsigned)n_pages;
            row = ((int64_t)(there ? page : 0) << shift) + (t0 & ((1 << shift) - 1));
            bytes = there ? bytes : 0;
        }
        return __builtin_amdgcn_make_buffer_rsrc(uniform_ptr(base + row * rb), 0, bytes, kRsrcWord3);
    }
};

// Fetches rows r0 .. r0 + 15 of a unit's queries into a tile in LDS (past the last row: the
// last again).
template <class P>
__device__ __forceinline__ void fetch_q(const WeightArgs &a, const WeightSeq &s, int b, int g, int r0, char *dst) {
    using T = typename P::QTile;
    r0 = min(r0, s.rows - 1);
    const int i0 = query_row(a, r0);
    const char *base = (const char *)a.q + (((int64_t)b * a.max_rows + i0) * a.n_head + g * a.gq) * P::q_bytes;
    const __amdgpu_buffer_rsrc_t rows = __builtin_amdgcn_make_buffer_rsrc(uniform_ptr(base), 0, 0x7fffffff, kRsrcWord3);
#pragma unroll
    for (int d = 0; d < T::N; d++) {
        const int r = min(r0 + T::row(d), s.rows - 1), i = query_row(a, r);
        dma16_cached(rows, dst + d * 1024, ((i - i0) * a.n_head + r - i * a.gq) * P::q_bytes + T::col(d), 0);
    }
}
// A tile of queries from LDS, as an operand (see Dot::make_q).
template <class P>
__device__ __forceinline__ float read_q(typename P::Q &q, const char *tile, bool neg) {
    typename P::Raw raw;
#pragma unroll
    for (int c = 0; c < P::QTile::N; c++) raw.x[c] = lds_read_b128(lds_addr(tile) + P::QTile::at(P::raw_chunk(c)));
    lds_wait(raw.x);
    return P::make_q(q, raw, neg);
}

constexpr int kWeightT = 256, kWeightW = 4;

// f(P::H tiles, their first key) over the steps of H tiles of keys k0 .. k1 - 1 (k0 a multiple
// of 32) that are this wave's, one of W, NB steps in flight in its ring.  f makes STORES stores (0: or none), which are counted with the
// loads and may be in flight as long as these.  start() is called behind the first loads.
template <class P, int NB, int W, int STORES, class S, class F>
__device__ __forceinline__ void each_step(const WeightArgs &a, const WeightSeq &s, int b, int g, int k0, int k1, int wave,
                                          char *ring, S &&start, F &&f) {
    using T = typename P::KTile;
    constexpr int H = P::H, N = 16 * H, step = N * W;
    int off[T::N];
    uint32_t at[P::KC];
#pragma unroll
    for (int d = 0; d < T::N; d++) off[d] = T::row(d) * (int)a.rb + T::col(d);
#pragma unroll
    for (int c = 0; c < P::KC; c++) at[c] = lds_addr(ring) + T::at(4 * c + ((threadIdx.x & 63) >> 4));
    for (int e0 = k0; e0 < k1; e0 = (e0 & -kWeightKeys) + kWeightKeys) {
        const int e1 = min(k1, (e0 & -kWeightKeys) + kWeightKeys), first = e0 + N * wave, last = (e1 - 1) & -N;
        const KeySource<P> src(a, s, b, g, e0);
        auto fetch = [&](int j, int t) __attribute__((always_inline)) {
            const __amdgpu_buffer_rsrc_t r = src.rows(t, N);
#pragma unroll
            for (int h = 0; h < H; h++)
#pragma unroll
                for (int d = 0; d < T::N; d++) {
                    char *dst = ring + j * P::step_bytes + h * T::bytes + d * 1024;
                    if (STORES) dma16(r, dst, off[d] + h * 16 * (int)a.rb, 0);
                    else dma16_cached(r, dst, off[d] + h * 16 * (int)a.rb, 0);
                }
        };
#pragma unroll
        for (int j = 0; j < NB; j++) fetch(j, min(first + step * j, last));
        if (e0 == k0) start();
        for (int t0 = first; t0 < e1; t0 += step * NB)
            static_for<0, NB>([&](auto J) __attribute__((always_inline)) {
                constexpr int j = decltype(J)::value;
                const int t = t0 + step * j;
                if (t >= e1) return;
                typename P::K k[H];
                // newer than this step's loads: NB - 1 steps' loads, and from the second round on NB
                // steps' stores
                constexpr int loads = (NB - 1) * H * T::N;
                if (STORES == 0 || t0 == first) vm_wait_n<loads>();
                else vm_wait_n<loads + NB * STORES>();
                static_for<0, H>([&](auto HH) __attribute__((always_inline)) {
                    constexpr int h = decltype(HH)::value;
#pragma unroll
                    for (int c = 0; c < P::KC; c++) k[h].x[c] = lds_read_b128_at<j * P::step_bytes + h * T::bytes>(at[c]);
                });
#pragma unroll
                for (int h = 0; h < H; h++) lds_wait(k[h].x);
                fetch(j, min(t + step * NB, last));
                f(k, t);
            });
        vm_wait_n<0>();  // (the ring is refilled, or given up)
    }
}

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// The lengths of a batch are on the device.  Where a call has few row blocks, all its
// sequences together are cut into up to spread + batch parts of one length, so that one round of
// workgroups is busy to its end: returns that length, and in lane b the parts of
// sequences 0 .. b (up to 64 of them).
__device__ __forceinline__ int weight_spread(const WeightArgs &a, int &upto) {
    const int lane = threadIdx.x & 63;
    int keys = 0;
    if (lane < a.batch) {
        const WeightSeq s(a, lane);
        int lo = 0, hi = 0;
        if (s.rows) s.keys(a, 0, s.rows, lo, hi);
        keys = max(0, hi - (lo & ~31));
    }
    // the shortest length, in steps of a sixteenth, that makes no more than spread + batch parts
    // (total / spread always does)
    const int total = __builtin_amdgcn_readlane(wave_scan(keys), 63), most = a.spread + a.batch;
    int chunk = max(128, (total / most + 127) & ~127);
    for (;; chunk += max(128, chunk / 16 & ~127)) {
        upto = wave_scan((keys + chunk - 1) / chunk);
        if (__builtin_amdgcn_readlane(upto, 63) <= most) return chunk;
    }
}
// The parts of a row block: part j has the keys from org + j chunk on; it is part
// first + j * step of the call.
struct WeightParts {
    int chunk, org, first, step;
};
__device__ __forceinline__ WeightParts weight_parts(const WeightArgs &a, const WeightSeq &s, int b, int g, int block, int lo, int chunk,
                                                    int upto) {
    WeightParts p{chunk, 0, 0, 1};
    if (!a.spread) {
        p.org = lo / chunk * chunk;
        p.first = ((b * a.n_kv + g) * a.blocks + block) * a.splits;
        return p;
    }
    int all_lo, all_hi;
    s.keys(a, 0, s.rows, all_lo, all_hi);
    p.org = all_lo & ~31;
    p.first = ((b ? __shfl(upto, b - 1) : 0) * a.blocks + block) * a.n_kv + g;
    p.step = a.blocks * a.n_kv;
    return p;
}

constexpr float kNoScore = -3e38f;  // a running maximum before any score

// Largest score and sum of RT * 16 rows over a part of their keys; the four waves
// take its tiles in turn.  STORE: and the scores.
template <class TQ, class TK, int D, int RT, bool STORE>
__global__ __launch_bounds__(kWeightT, (Dot<TQ, TK, D>::waves)) void weight_rows_kernel(WeightArgs a) {
    using P = Dot<TQ, TK, D>;
    constexpr int H = P::H, NB = P::KC <= 2 ? 4 : 2;
    // the queries come through the ring, or where there is room beside it while it fills
    constexpr bool APART = RT == 1 && P::QTile::bytes <= 8192;
    static_assert(RT * P::QTile::bytes <= kWeightW * NB * P::step_bytes, "queries in the ring");
    __shared__ __attribute__((aligned(1024))) char ring[kWeightW][NB * P::step_bytes];
    __shared__ __attribute__((aligned(1024))) char apart[APART ? P::QTile::bytes : 16];
    __shared__ float2 join[kWeightW][RT * 16];
    __shared__ int pos[RT * 16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int b, g, block, split, chunk = a.chunk;
    if (a.spread) {
        int upto;
        chunk = weight_spread(a, upto);
        const int slot = blockIdx.x / (a.n_kv * a.blocks);
        b = __popcll(__ballot(upto <= slot));
        if (b >= a.batch) return;
        split = slot - (b ? __builtin_amdgcn_readlane(upto, b - 1) : 0);
        g = blockIdx.x % a.n_kv, block = blockIdx.x / a.n_kv % a.blocks;
    } else {
        const int unit = blockIdx.x % a.units, rest = blockIdx.x / a.units;  // (what shares keys on one XCD)
        split = rest % a.splits, block = a.blocks - 1 - rest / a.splits, b = unit / a.n_kv, g = unit % a.n_kv;
    }
    const int unit = b * a.n_kv + g, r0 = block * RT * 16;
    const WeightSeq s(a, b);
    const int r1 = min(r0 + RT * 16, s.rows);
    if (r0 >= r1) return;
    int lo, hi;
    s.keys(a, r0, r1, lo, hi);
    int org = lo / chunk * chunk;
    if (a.spread) {
        int all_lo, all_hi;
        s.keys(a, 0, s.rows, all_lo, all_hi);
        org = all_lo & ~31;
    }
    const int k0 = max(lo & ~31, org + split * chunk), k1 = min(hi, org + (split + 1) * chunk);
    if (k0 >= k1) return;
    // a row at position p sees the keys t with 0 <= p - t < span
    const unsigned span = a.window ? a.window : INT_MAX;
    const int score_tile = a.rows_pad * 16;
    const float aqs = fabsf(a.qs);
    float *const score = STORE ? a.score + (unit * a.tiles * a.rows_pad + (lane & 15)) * 16 + 4 * (lane >> 4) : nullptr;
    typename P::Q q[RT];
    float row_qs[P::NP == 2 ? RT : 1], m[RT], l[RT];
    auto qs = [&](int i) __attribute__((always_inline)) { return P::NP == 2 ? row_qs[P::NP == 2 ? i : 0] : aqs; };
    char *const staged = APART ? apart : ring[0];
    auto load_q = [&](auto behind) __attribute__((always_inline)) {  // behind: newer loads than the queries'
        vm_wait_n<decltype(behind)::value>();
        __syncthreads();
#pragma unroll
        for (int i = 0; i < RT; i++) {
            const float back = read_q<P>(q[i], staged + i * P::QTile::bytes, a.qs < 0.f);
            if (P::NP == 2) row_qs[P::NP == 2 ? i : 0] = fmaxf(aqs * back, 1.17549435e-38f);  // (not 0: see a.qs)
            m[i] = kNoScore, l[i] = 0.f;
        }
    };
    if (tid < RT * 16) pos[tid] = r0 + tid < s.rows ? s.first + query_row(a, r0 + tid) : -1;
    if (wave < RT) fetch_q<P>(a, s, b, g, r0 + wave * 16, staged + wave * P::QTile::bytes);
    if (!APART) {
        load_q(Int<0>{});
        __syncthreads();
    }
    auto start = [&]() __attribute__((always_inline)) {
        if (APART) load_q(Int<NB * H * P::KTile::N>{});
    };
    // tiles that every row sees whole
    const int all_lo = a.window ? s.first + query_row(a, r1 - 1) + 1 - a.window : 0, all_hi = s.first + query_row(a, r0) + 1;
    auto tiles = [&](const typename P::K *k, int t0, auto mask) __attribute__((always_inline)) {
        f32x4 x[RT][H];
        P::template dots<false>(x, k, q);
#pragma unroll
        for (int i = 0; i < RT; i++) {
            if constexpr (mask.value) {
                const int d = pos[i * 16 + (lane & 15)] - t0 - 4 * (lane >> 4);  // keys up to d are seen
#pragma unroll
                for (int j = 0; j < 4 * H; j++) {
                    const int t = (j & 3) + (j >> 2) * 16;
                    if ((unsigned)(d - t) >= span) x[i][j >> 2][j & 3] = -INFINITY;
                }
            }
            if constexpr (STORE) {
                if ((lane & 15) < s.rows)
#pragma unroll
                    for (int h = 0; h < H; h++)
                        *(f32x4 *)(score + ((t0 >> 4) + h) * (int64_t)score_tile) =
                            x[i][h] * qs(i);
            }
            float top = -INFINITY, e[4 * H], add[H];
#pragma unroll
            for (int j = 0; j < 4 * H; j++) top = fmaxf(top, x[i][j >> 2][j & 3]);
            const float up = fmaxf(m[i], top * qs(i)), back = exp2_of(m[i] - up);
            m[i] = up;
#pragma unroll
            for (int j = 0; j < 4 * H; j++) e[j] = exp2_of(fmaf(x[i][j >> 2][j & 3], qs(i), -up));
#pragma unroll
            for (int h = 0; h < H; h++) add[h] = (e[4 * h] + e[4 * h + 1]) + (e[4 * h + 2] + e[4 * h + 3]);
            l[i] = fmaf(l[i], back, add[0] + (H > 1 ? add[H - 1] : 0.f));
        }
    };
    each_step<P, NB, kWeightW, STORE ? H : 0>(a, s, b, g, k0, k1, wave, ring[wave], start, [&](const typename P::K *k, int t0) __attribute__((always_inline)) {
        if (t0 >= all_lo && t0 + 16 * H <= all_hi) tiles(k, t0, Int<0>{});
        else tiles(k, t0, Int<1>{});
    });
#pragma unroll
    for (int i = 0; i < RT; i++) {
        const float top = rows_max(m[i]);
        const float sum = rows_sum(l[i] * exp2_of(m[i] - top));
        if (lane < 16) join[wave][i * 16 + lane] = float2{top, sum};
    }
    __syncthreads();
    if (tid < (a.direct ? RT * 16 : r1 - r0)) {
        float top = join[0][tid].x, sum = 0.f;
        for (int w = 1; w < kWeightW; w++) top = fmaxf(top, join[w][tid].x);
        for (int w = 0; w < kWeightW; w++) sum += join[w][tid].y * exp2_of(join[w][tid].x - top);
        if (a.direct) {  // (past the last row: weights of 0)
            const float lse = tid < r1 - r0 && sum != 0.f ? top + __builtin_amdgcn_logf(sum) : INFINITY;
            a.lse[(int64_t)unit * a.rows_pad + r0 + tid] = float2{lse, aqs};
            return;
        }
        const int part = a.spread ? (int)blockIdx.x : (unit * a.blocks + block) * a.splits + split;
        a.ml[(int64_t)part * RT * 16 + tid] = float2{top, sum};
    }
    if (P::NP == 2 && !STORE && k0 == max(lo & ~31, org) && wave == 0 && lane < 16)
#pragma unroll
        for (int i = 0; i < RT; i++) a.row_qs[(int64_t)unit * a.rows_pad + r0 + i * 16 + lane] = qs(i);
}

// log2 of a row's denominator from its parts, by 16 lanes; +inf where it sees nothing
// (its weights are then 2^-inf).  upto: of weight_spread, in every lane of the wave.
__device__ __forceinline__ float row_lse(const WeightArgs &a, const WeightSeq &s, int b, int g, int r, int block_rows, int chunk,
                                         int upto) {
    const int block = r / block_rows, r0 = block * block_rows;
    int lo = 0, hi = 0;
    if (r < s.rows) s.keys(a, r0, min(r0 + block_rows, s.rows), lo, hi);
    const WeightParts p = weight_parts(a, s, b, g, block, lo, chunk, upto);
    float m = kNoScore, l = 0.f;
    if (hi > lo) {
        const int last = (hi - 1 - p.org) / chunk;
        for (int j = (lo - p.org) / chunk + (threadIdx.x & 15); j <= last; j += 16) {
            const float2 x = a.ml[(int64_t)(p.first + j * p.step) * block_rows + r - r0];
            const float up = fmaxf(m, x.x);
            l = l * exp2_of(m - up) + x.y * exp2_of(x.x - up);
            m = up;
        }
    }
    float top = m;
    top = fmaxf(top, dpp<kDppXor1>(top)), top = fmaxf(top, dpp<kDppXor2>(top));
    top = fmaxf(top, dpp<kDppHalfMirror>(top)), top = fmaxf(top, dpp<kDppMirror>(top));
    l = group_sum<16>(l * exp2_of(m - top));
    return l == 0.f ? INFINITY : top + __builtin_amdgcn_logf(l);
}

// The denominators of all rows, 16 lanes a row.
__global__ __launch_bounds__(256) void weight_merge_kernel(WeightArgs a, int block_rows, int scaled) {
    const int64_t at = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4), all = (int64_t)a.units * a.rows_pad;
    int upto = 0, chunk = a.chunk;
    if (a.spread) chunk = weight_spread(a, upto);
    const int unit = (int)(min(at, all - 1) / a.rows_pad), r = (int)(min(at, all - 1) % a.rows_pad);
    const WeightSeq s(a, unit / a.n_kv);
    const float lse = row_lse(a, s, unit / a.n_kv, unit % a.n_kv, r, block_rows, chunk, upto);
    if (at < all && (threadIdx.x & 15) == 0)
        a.lse[at] = float2{lse, scaled && lse != INFINITY ? a.row_qs[at] : fabsf(a.qs)};
}

__device__ __forceinline__ void put_weight(const WeightArgs &a, int unit, int t, float sum) {
    float *w = a.w + (int64_t)unit * a.w_stride + t;
    *w = a.decay == 0.f ? sum : fmaf(a.decay, *w, sum);
}

// Stored scores of up to 16 rows: a thread four keys, whose scores and old weights are
// on their way while the denominators are found.
__global__ __launch_bounds__(kWeightT) void weight_sums_kernel(WeightArgs a) {
    __shared__ float lse[16];
    const int tid = threadIdx.x, unit = blockIdx.x % a.units, t0 = (blockIdx.x / a.units * kWeightT + tid) * 4;
    const int b = unit / a.n_kv;
    const WeightSeq s(a, b);
    if ((int)(blockIdx.x / a.units) * kWeightT * 4 >= s.len) return;
    int lo = 0, hi = 0;
    if (s.rows) s.keys(a, 0, s.rows, lo, hi);
    const bool stored = t0 < hi && t0 + 3 >= (lo & ~31);  // (whole tiles were)
    const float *x = a.score + (unit * a.tiles + (stored ? t0 >> 4 : 0)) * a.rows_pad * 16 + (t0 & 15);
    float *w = a.w + (int64_t)unit * a.w_stride + t0;
    f32x4 v[16], sum{};
    float old[4];
#pragma unroll
    for (int r = 0; r < 16; r++)
        if (r < s.rows && stored) v[r] = *(const f32x4 *)(x + r * 16);
#pragma unroll
    for (int j = 0; j < 4; j++) old[j] = a.decay != 0.f && t0 + j < s.len ? w[j] : 0.f;
    int upto = 0, chunk = a.chunk;
    if (a.spread) chunk = weight_spread(a, upto);
    const float mine = row_lse(a, s, b, unit % a.n_kv, min(tid >> 4, a.rows_pad - 1), 16, chunk, upto);
    if ((tid & 15) == 0) lse[tid >> 4] = mine;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 16; r++)
        if (r < s.rows && stored)
#pragma unroll
            for (int j = 0; j < 4; j++) sum[j] += exp2_of(v[r][j] - lse[r]);
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (t0 + j < s.len) w[j] = a.decay == 0.f ? sum[j] : fmaf(a.decay, old[j], sum[j]);
}

// Weights of up to RS * RT * 16 rows, which stay in registers, over streamed keys: RS waves
// share a step's keys, each with its own rows; their sums meet in LDS at the end.
template <class TQ, class TK, int D, int RT, int RS>
__global__ __launch_bounds__(kWeightT, (Dot<TQ, TK, D>::waves)) void weight_stream_kernel(WeightArgs a) {
    using P = Dot<TQ, TK, D>;
    constexpr int W = kWeightW / RS, rows = RS * RT * 16;
    constexpr int NB = P::KC <= 2 ? 4 : 2;
    __shared__ __attribute__((aligned(1024))) char ring[kWeightW][NB * P::step_bytes];
    static_assert(RS * RT * P::QTile::bytes <= kWeightW * NB * P::step_bytes, "queries in the ring");
    __shared__ float sums[RS][kWeightKeys / RS];
    constexpr int H = P::H;
    __shared__ int pos[rows];
    __shared__ float lse[rows], row_qs[rows];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int unit = blockIdx.x % a.units, rest = blockIdx.x / a.units, b = unit / a.n_kv, g = unit % a.n_kv;
    const WeightSeq s(a, b);
    const int chunk = min(a.chunk, kWeightKeys / RS), k0 = rest * chunk, k1 = min(s.len, k0 + chunk), i0 = wave % RS * RT;
    if (k0 >= k1) return;
    int lo = 0, hi = 0;
    if (s.rows) s.keys(a, 0, s.rows, lo, hi);
    if (k0 >= hi || k1 <= lo) {  // no row sees these
        for (int t = k0 + tid; t < k1; t += kWeightT) put_weight(a, unit, t, 0.f);
        return;
    }
    const unsigned span = a.window ? a.window : INT_MAX;
    const float aqs = fabsf(a.qs);
    typename P::Q q[RT];
    if (tid < rows) {
        const float2 x = a.lse[(int64_t)unit * a.rows_pad + tid];
        lse[tid] = x.x, row_qs[tid] = x.y;
        pos[tid] = x.x == INFINITY ? -1 : s.first + query_row(a, tid);  // (also where there is no row)
    }
    for (int i = wave; i < RS * RT; i += kWeightW) fetch_q<P>(a, s, b, g, i * 16, ring[0] + i * P::QTile::bytes);
    vm_wait_n<0>();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RT; i++) read_q<P>(q[i], ring[0] + (i0 + i) * P::QTile::bytes, a.qs < 0.f);
    __syncthreads();
    auto start = [] {};
    const int all_lo = a.window ? s.first + query_row(a, s.rows - 1) + 1 - a.window : 0, all_hi = s.first + 1;
    auto tiles = [&](const typename P::K *k, int t0, auto mask) __attribute__((always_inline)) {
        f32x4 x[RT][H];
        float sum[H];
        P::template dots<true>(x, k, q);
#pragma unroll
        for (int i = 0; i < RT; i++) {
            const int r = (i0 + i) * 16 + 4 * (lane >> 4);  // the lane's four rows
            const f32x4 ls = *(const f32x4 *)(lse + r);
            f32x4 qs;
            if (P::NP == 2) qs = *(const f32x4 *)(row_qs + r);
            int ps[4];
            if (mask.value) {
                const int4 p = *(const int4 *)(pos + r);
                ps[0] = p.x, ps[1] = p.y, ps[2] = p.z, ps[3] = p.w;
            }
#pragma unroll
            for (int h = 0; h < H; h++) {
                float e[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    e[j] = exp2_of(fmaf(x[i][h][j], P::NP == 2 ? qs[j] : aqs, -ls[j]));
                    const int t = t0 + 16 * h + (lane & 15);
                    if (mask.value && (unsigned)(ps[j] - t) >= span) e[j] = 0.f;
                }
                const float add = (e[0] + e[1]) + (e[2] + e[3]);
                sum[h] = i ? sum[h] + add : add;
            }
        }
#pragma unroll
        for (int h = 0; h < H; h++) {
            sum[h] = rows_sum(sum[h]);
            if (lane < 16) sums[wave % RS][t0 - k0 + 16 * h + lane] = sum[h];
        }
    };
    each_step<P, NB, W, 0>(a, s, b, g, k0, k1, wave / RS, ring[wave], start, [&](const typename P::K *k, int t0) __attribute__((always_inline)) {
        if (t0 >= all_lo && t0 + 16 * H <= all_hi) tiles(k, t0, Int<0>{});
        else tiles(k, t0, Int<1>{});
    });
    __syncthreads();
    for (int t = k0 + tid; t < k1; t += kWeightT) {
        float all = sums[0][t - k0];
#pragma unroll
        for (int i = 1; i < RS; i++) all += sums[i][t - k0];
        put_weight(a, unit, t, all);
    }
}

// Sums of the weights of KT * 16 keys, which stay in registers, over row_chunk streamed
// rows; the four waves take row tiles in turn, the next one in flight.
template <class TQ, class TK, int D>
__global__ __launch_bounds__(kWeightT, (Dot<TQ, TK, D>::keys_waves)) void weight_keys_kernel(WeightArgs a) {
    using P = Dot<TQ, TK, D>;
    using T = typename P::QTile;
    constexpr int KT = P::kt, NB = 2, R = 16 * kWeightW, stage = T::bytes + 1024;  // the rows, their (lse, qs)
    static_assert(KT * P::KTile::bytes <= kWeightW * NB * stage, "keys in the ring");
    __shared__ __attribute__((aligned(1024))) char ring[kWeightW][NB * stage];
    __shared__ float join[kWeightW][KT * 16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int unit = blockIdx.x % a.units, rest = blockIdx.x / a.units, part = rest % a.parts, b = unit / a.n_kv, g = unit % a.n_kv;
    const int k0 = rest / a.parts * KT * 16;
    const WeightSeq s(a, b);
    const int k1 = min(k0 + KT * 16, s.len);
    if (k0 >= k1) return;
    // rows that see any of the keys
    const int lo = max(part * a.row_chunk, max(0, k0 - s.first) * a.gq) & ~15;
    int hi = min(s.rows, (part + 1) * a.row_chunk);
    if (a.window) hi = (int)min((int64_t)hi, (int64_t)max(0, k1 - 1 + a.window - s.first) * a.gq);
    float *out = a.part + ((int64_t)part * a.units + unit) * a.max_len;
    if (lo >= hi) {
        for (int t = k0 + tid; t < k1; t += kWeightT) out[t] = 0.f;
        return;
    }
    const int window = a.window;
    const unsigned span = window ? window : INT_MAX;
    const float aqs = fabsf(a.qs);
    uint32_t at[T::N];
#pragma unroll
    for (int c = 0; c < T::N; c++) at[c] = lds_addr(ring[wave]) + T::at(P::raw_chunk(c));
    const uint32_t at_ls = lds_addr(ring[wave]) + T::bytes + (lane >> 4) * 32;
    auto fetch = [&](int j, int r0) __attribute__((always_inline)) {
        char *dst = ring[wave] + j * stage;
        fetch_q<P>(a, s, b, g, r0, dst);
        // (lse, qs) of 16 rows in the first 8 lanes; past them nothing is read
        const __amdgpu_buffer_rsrc_t ls =
            __builtin_amdgcn_make_buffer_rsrc(uniform_ptr(a.lse + (int64_t)unit * a.rows_pad + r0), 0, 128, kRsrcWord3);
        dma16_cached(ls, dst + T::bytes, lane * 16, 0);
    };
    typename P::K k[KT];
    float sum[KT];
#pragma unroll
    for (int i = 0; i < KT; i++) sum[i] = 0.f;
    auto tile = [&](const typename P::Q &q, const f32x4 (&w)[2], int r0, auto mask) __attribute__((always_inline)) {
        const float lse[4] = {w[0][0], w[0][2], w[1][0], w[1][2]}, qs[4] = {w[0][1], w[0][3], w[1][1], w[1][3]};
        int pos[4];
        if constexpr (mask.value)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int r = r0 + 4 * (lane >> 4) + j;
                pos[j] = r < s.rows && lse[j] != INFINITY ? s.first + query_row(a, r) : -1;
            }
        constexpr int G = KT < 4 ? KT : 4;
#pragma unroll
        for (int i0 = 0; i0 < KT; i0 += G) {
            f32x4 x[1][G];
            P::template dots<true>(x, k + i0, &q);
#pragma unroll
            for (int i = 0; i < G; i++) {
                float e[4];
#pragma unroll
                for (int j = 0; j < 4; j++) e[j] = exp2_of(fmaf(x[0][i][j], P::NP == 2 ? qs[j] : aqs, -lse[j]));
                if constexpr (mask.value) {
                    const int t = k0 + 16 * (i0 + i) + (lane & 15);
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if ((unsigned)(pos[j] - t) >= span) e[j] = 0.f;
                }
                sum[i0 + i] += (e[0] + e[1]) + (e[2] + e[3]);
            }
        }
    };
    const int last = (hi - 1) & ~15;
    {  // the keys, through the ring
        using KT_ = typename P::KTile;
        const KeySource<P> src(a, s, b, g, k0);
        for (int i = wave; i < KT; i += kWeightW) {
            const __amdgpu_buffer_rsrc_t rsrc = src.rows(min(k0 + 16 * i, (k1 - 1) & ~15), 16);
#pragma unroll
            for (int d = 0; d < KT_::N; d++)
                dma16_cached(rsrc, ring[0] + i * KT_::bytes + d * 1024, KT_::row(d) * (int)a.rb + KT_::col(d), 0);
        }
        vm_wait_n<0>();
        __syncthreads();
#pragma unroll
        for (int i = 0; i < KT; i++) {
#pragma unroll
            for (int c = 0; c < P::KC; c++)
                k[i].x[c] = lds_read_b128(lds_addr(ring[0]) + i * KT_::bytes + KT_::at(4 * c + (lane >> 4)));
            lds_wait(k[i].x);
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < NB; j++) fetch(j, min(lo + 16 * wave + j * R, last));
    for (int r0 = lo + 16 * wave; r0 < hi; r0 += NB * R)
        static_for<0, NB>([&](auto J) __attribute__((always_inline)) {
            constexpr int j = decltype(J)::value;
            const int r = r0 + j * R;
            if (r >= hi) return;
            typename P::Raw raw;
            u32x4 ls[2];
            vm_wait_n<(NB - 1) * (T::N + 1)>();
#pragma unroll
            for (int c = 0; c < T::N; c++) raw.x[c] = lds_read_b128_at<j * stage>(at[c]);
            ls[0] = lds_read_b128_at<j * stage>(at_ls), ls[1] = lds_read_b128_at<j * stage + 16>(at_ls);
            lds_wait(raw.x);
            tie(ls[0]), tie(ls[1]);
            fetch(j, min(r + NB * R, last));
            typename P::Q q;
            P::make_q(q, raw, a.qs < 0.f);
            const f32x4 w[2] = {__builtin_bit_cast(f32x4, ls[0]), __builtin_bit_cast(f32x4, ls[1])};
            const int p0 = s.first + query_row(a, r), p1 = s.first + query_row(a, min(r + 16, s.rows) - 1);
            if (k0 + KT * 16 - 1 <= p0 && (!window || k0 > p1 - window)) tile(q, w, r, Int<0>{});
            else tile(q, w, r, Int<1>{});
        });
    vm_wait_n<0>();
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
// Which way (us, scores stored / computed again, bf16 x 128): 8 sequences of 16K, 8 rows of a
// kv head 77 / 103, 16 rows 85 / 103; of 4K-32K, 8 rows 53 / 81; one of 32K 20.6 / 28.6.
// Sequences cut together / each alone: 4K-32K 53 / 56, one of 32K 19.5 / 23.8, equal lengths
// the same.
struct WeightCut {
    int rt, mode;  // row tiles of a wave; 0: scores stored, 1: rows in registers, 2: keys in registers
    int rows_pad, blocks, chunk, splits, spread, row_chunk, parts;
    int64_t wgs;  // of weight_rows_kernel, its parts
    size_t ml, qs, lse, score, part, bytes;  // offsets
};
// Registers of a row tile, and the most of them in a wave (Dot::q_regs, Dot::rt).
static int weight_q_regs(int q_dtype, int dtype, int D) {
    return D * dtype_bytes(dtype) / 16 * (q_dtype == dtype ? 1 : dtype == ULLM_DT_F16 ? 2 : 3);
}
static int weight_rt(int regs) { return regs <= 16 ? 4 : regs <= 48 ? 2 : 1; }
// Workgroups aimed at where row blocks are many: a 2048-token prompt takes 32.5 us in its rows
// with 512 or 1024, 43.5 with 2048, 60 with 4096 (a start each).
constexpr int64_t kWeightWgs = 1024;
static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
static WeightCut weight_cut(int q_dtype, int dtype, int64_t batch, int max_rows, int max_len, int window, int n_head,
                            int64_t n_kv, int D) {
    WeightCut c{};
    const int64_t rows = (int64_t)max_rows * (n_head / n_kv), units = batch * n_kv;
    const int regs = weight_q_regs(q_dtype, dtype, D), top = weight_rt(regs);
    c.rt = 1;
    while (c.rt < top && c.rt * 16 < rows) c.rt *= 2;
    c.blocks = (int)((rows + c.rt * 16 - 1) / (c.rt * 16));
    c.mode = rows <= 16 ? 0 : rows <= kWeightW * top * 16 ? 1 : 2;
    c.rows_pad = c.mode == 0 ? (int)rows : (int)((rows + 255) / 256 * 256);
    // parts of a row block's keys, whole tiles for every wave
    const int64_t keys = window > 0 && window < max_len ? std::min<int64_t>(max_len, (int64_t)window + max_rows) : max_len;
    const int64_t want = (keys * units * c.blocks + kWeightWgs - 1) / kWeightWgs;
    c.chunk = (int)std::max<int64_t>(std::min<int64_t>((want + 127) / 128, (max_len + 127) / 128) * 128, 128);
    c.splits = (int)((keys + c.chunk - 1) / c.chunk + (window > 0 ? 1 : 0));
    c.wgs = units * c.blocks * c.splits;
    // one sequence's keys or those of up to 64 together: one round of the card
    if (c.mode <= 1 && batch <= 64 && batch * max_len <= INT_MAX) {
        const int64_t each = n_kv * c.blocks, round = D * dtype_bytes(dtype) > 512 ? 256 : 512;
        c.spread = (int)std::max<int64_t>(round / each - batch, std::max<int64_t>(batch, 1));
        c.wgs = (c.spread + batch) * each;
    }
    // (8192 rows of a kv head over 2048 keys, the whole call: 69 us in 8 parts, 70 in 6, 81 in 4, 83 in 2)
    c.parts = (int)std::min<int64_t>(8, (rows + 511) / 512);
    // (fewer where the key blocks, of 32 keys or more, alone come near the 2^24 workgroups of a grid)
    const int64_t key_blocks = units * ((max_len + 31) / 32);
    while (c.parts > 1 && key_blocks * c.parts >= 1 << 24) c.parts--;
    c.row_chunk = (int)(((rows + c.parts - 1) / std::max(c.parts, 1) + 63) / 64 * 64);
    size_t at = 0;
    const size_t entries = (size_t)units * c.rows_pad;
    c.ml = at, at += up256((size_t)c.wgs * c.rt * 16 * sizeof(float2));
    c.qs = at, at += up256(entries * sizeof(float));
    c.lse = at, at += c.mode ? up256(entries * sizeof(float2)) : 0;
    c.score = at, at += c.mode == 0 ? up256((size_t)units * ((max_len + 31) / 32) * c.rows_pad * 32 * sizeof(float)) : 0;
    c.part = at, at += c.mode == 2 ? up256((size_t)c.parts * units * max_len * sizeof(float)) : 0;
    c.bytes = at;
    return c;
}

template <class TQ, class TK, int D, int RT, int RS>
static void launch_stream(const WeightArgs &a, hipStream_t st) {
    const int chunk = std::min(a.chunk, kWeightKeys / RS);
    if constexpr (RT <= Dot<TQ, TK, D>::rt)
        launch_kernel(weight_stream_kernel<TQ, TK, D, RT, RS>, dim3(a.units * ((a.max_len + chunk - 1) / chunk)), dim3(kWeightT), 0, st, a);
}
template <class TQ, class TK, int D, int RT>
static void launch_rows(const WeightArgs &a, unsigned wgs, hipStream_t st) {
    if constexpr (RT <= Dot<TQ, TK, D>::rt)
        launch_kernel(weight_rows_kernel<TQ, TK, D, RT, false>, dim3(wgs), dim3(kWeightT), 0, st, a);
}
template <class TQ, class TK, int D>
static void launch_weights(const WeightArgs &a, const WeightCut &c, hipStream_t st) {
    using P = Dot<TQ, TK, D>;
    const dim3 wg(kWeightT);
    const unsigned units = a.units;
    if (c.mode == 0) {
        launch_kernel(weight_rows_kernel<TQ, TK, D, 1, true>, dim3((unsigned)c.wgs), wg, 0, st, a);
        launch_kernel(weight_sums_kernel, dim3(units * ((a.max_len + 4 * kWeightT - 1) / (4 * kWeightT))), wg, 0, st, a);
        return;
    }
    if (c.rt == 1) launch_rows<TQ, TK, D, 1>(a, c.wgs, st);
    else if (c.rt == 2) launch_rows<TQ, TK, D, 2>(a, c.wgs, st);
    else launch_rows<TQ, TK, D, 4>(a, c.wgs, st);
    if (!a.direct) launch_kernel(weight_merge_kernel, dim3(((size_t)units * c.rows_pad + 15) / 16), dim3(256), 0, st, a, c.rt * 16, (int)(P::NP == 2));
    if (c.mode == 1) {
        // as few waves to a key as hold the rows
        const int tiles = (a.max_rows * a.gq + 15) / 16;
        if (tiles <= 2 && P::rt >= 2) launch_stream<TQ, TK, D, 2, 1>(a, st);
        else if (tiles <= 4 && P::rt >= 4) launch_stream<TQ, TK, D, 4, 1>(a, st);
        else if (tiles <= 2 * P::rt) launch_stream<TQ, TK, D, P::rt, 2>(a, st);
        else launch_stream<TQ, TK, D, P::rt, 4>(a, st);
        return;
    }
    constexpr int keys = P::kt * 16;
    launch_kernel(weight_keys_kernel<TQ, TK, D>, dim3(units * a.parts * ((a.max_len + keys - 1) / keys)), wg, 0, st, a);
    launch_kernel(weight_join_kernel, dim3(units * ((a.max_len + kWeightT - 1) / kWeightT)), wg, 0, st, a);
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
    if (kv_stride < (int64_t)a.n_kv * head_dim || kv_stride > INT_MAX / 256 || a.w_stride < a.max_len)
        return set_error(ULLM_HIP_E_INVALID, "%s: bad kv_stride, or weights_stride too small", fn);
    if (a.batch == 0 || a.max_len == 0) return ULLM_HIP_OK;
    if ((!a.q && a.max_rows) || !a.k || !a.len || !a.w) return set_error(ULLM_HIP_E_INVALID, "%s: null tensor pointer", fn);
    const int eb = dtype_bytes(dtype);
    if (((uintptr_t)a.q | (uintptr_t)a.k) & 15 || kv_stride * eb % 16 || a.seq_b % 16)
        return set_error(ULLM_HIP_E_INVALID, "%s: tensors and row strides must be 16-byte aligned", fn);
    const int rows = std::max(a.max_rows, 1);  // (none: the weights fade, as n_rows of 0 does)
    const WeightCut c = weight_cut(q_dtype, dtype, a.batch, rows, a.max_len, a.window, a.n_head, a.n_kv, head_dim);
    const int64_t units = (int64_t)a.batch * a.n_kv;
    // (a grid has less than 2^32 threads)
    if (c.wgs >= 1 << 24 || units * c.blocks * c.splits >= 1 << 30 || units * c.rows_pad >= 1 << 28 || units * ((a.max_len + 31) / 32) * c.parts >= 1 << 24)
        return set_error(ULLM_HIP_E_INVALID, "%s: too many rows or keys", fn);
    if (!ws || ws_bytes < c.bytes || (uintptr_t)ws & 255)
        return set_error(ULLM_HIP_E_WORKSPACE, "%s: workspace of %zu bytes, 256-byte aligned, needed", fn, c.bytes);
    a.gq = a.n_head / a.n_kv;
    a.gq_shift = 31 - __builtin_clz(a.gq);
    a.gq_mul = a.gq & (a.gq - 1) ? (uint32_t)((1ull << (32 + a.gq_shift)) / a.gq + 1) : 0;
    // (a scale of 0 as the least normal number: 0 times a masked score of -inf is none)
    a.qs = std::copysign(std::max(std::fabs(scale * kLog2e), 1.17549435e-38f), scale);
    a.rb = kv_stride * eb;
    a.units = (int)units, a.rows_pad = c.rows_pad, a.blocks = c.blocks, a.chunk = c.chunk, a.splits = c.splits, a.spread = c.spread;
    a.direct = c.mode == 2 && c.splits == 1 && (q_dtype == dtype || dtype != ULLM_DT_F16);
    a.row_chunk = c.row_chunk, a.parts = c.parts, a.tiles = (a.max_len + 31) / 32 * 2;
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
                       nullptr, 0, 0, 0, seq_lens, n_rows, max_rows, max_len, window, batch, n_head, n_kv_head, 0, 0, 0, 0.f,
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
                       seq_lens, n_rows, max_rows, max_len, window, batch, n_head, n_kv_head, 0, 0, 0, 0.f, decay, weights,
                       weights_stride};
    return key_weights("key_weights_paged", a, q_dtype, kv_dtype, kv_stride, head_dim, scale, workspace,
                       workspace_bytes, stream);
}

extern "C" size_t ullm_hip_key_weights_workspace_bytes(int kv_dtype, int batch, int max_rows, int max_len, int window,
                                                       int n_head, int n_kv_head, int head_dim) {
    if (!dtype_ok(kv_dtype) || (head_dim != 64 && head_dim != 128 && head_dim != 256) || batch < 1 || max_rows < 0 ||
        max_len < 1 || max_len > 1 << 30 || window < 0 || n_head < 1 || n_kv_head < 1 || n_head % n_kv_head || n_head > 65535 ||
        (int64_t)max_rows * n_head > 1 << 23)
        return 0;
    max_rows = std::max(max_rows, 1);  // (a call without rows is planned as one of one row)
    // For every call with fewer sequences, rows and positions too: parts of row blocks are at most
    // kWeightWgs and three more a block; the scores are those of up to 16 rows.
    const int gq = n_head / n_kv_head;
    const int64_t rows = (int64_t)max_rows * gq, units = (int64_t)batch * n_kv_head;
    size_t most = 0;
    for (int q_dtype : {(int)ULLM_DT_F32, kv_dtype}) {
        const int block = 16 * weight_rt(weight_q_regs(q_dtype, kv_dtype, head_dim));
        const int64_t blocks = (rows + block - 1) / block, pad = (rows + 255) / 256 * 256;
        size_t n = up256((kWeightWgs + 3 * units * blocks) * block * sizeof(float2)) + 2 * up256(units * pad * sizeof(float2));
        n += std::max((size_t)(gq <= 16 ? up256((size_t)units * ((max_len + 31) / 32) * std::min<int64_t>(rows, 16) * 32 * sizeof(float)) : 0),
                      up256((size_t)std::min<int64_t>(8, (rows + 511) / 512) * units * max_len * sizeof(float)));
        most = std::max(most, n);
    }
    return most;
}
