// A KV cache cut down to a budget by the attention weight that its positions
// have collected: ullm_hip_kv_evict(_paged).  Two launches: which positions of
// each layer, sequence and group of columns stay, then their rows moved together.
#include <algorithm>
#include <climits>
#include "common.hpp"
#include "wave.hpp"

namespace ullm {

struct EvictArgs {
    char *k, *v;
    int64_t rb, seq_b, layer_b;  // bytes of a row, from sequence to sequence, from layer to layer
    const int32_t *tab;          // null: contiguous
    int tab_stride, shift, n_pages, n_ctx;  // n_ctx: rows that a sequence can have
    const float *score;
    float *score_out;
    int64_t score_stride;
    const int32_t *len, *budget;
    int max_budget, sink, recent, groups, batch;
    int cols, one;  // 16-byte columns of a group; K and V are the same memory, which moves once
    int32_t *kept, *len_out;
};

// What stays of sequence b: n of its len positions, the first ones, the last ones
// and `best` of those between.
struct EvictSeq {
    int len, n, first, last, best;
    __device__ EvictSeq(const EvictArgs &a, int b) {
        len = min(max(a.len[b], 0), a.n_ctx);
        n = min(len, min(max(a.budget[b], 0), a.max_budget));
        first = min(a.sink, n);
        last = min(a.recent, n - first);
        best = n - first - last;
    }
};

constexpr int kPickT = 1024, kPickBins = 2048;

// Order of the weights as whole numbers: NaN below everything, -0 as 0.
__device__ __forceinline__ uint32_t score_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    if (x != x) return 0;
    return u >> 31 ? ~u : u | 0x80000000u;
}

// Inclusive sum of v over the workgroup, and the total; tmp: one word a wave.
__device__ __forceinline__ int pick_scan(int v, int *tmp, int &total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int x = wave_scan(v);
    __syncthreads();
    if (lane == 63) tmp[w] = x;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kPickT / 64; i++) {
        if (i < w) before += tmp[i];
        total += tmp[i];
    }
    return before + x;
}

// The best-th largest of the keys between first and len - last: bins of equal
// width over the range that still holds it (the keys' own smallest to largest
// at first: 2048 bins over floats as whole numbers are about a hundred to an
// octave, so that few lanes meet in a bin), until a bin holds one value or
// exactly as many keys as are wanted.  Then one pass in order writes what stays.
// Up to TILES * 4096 scores stay in registers, four neighbours a thread (more are read
// anew in each pass): bound by the barriers of three to four passes.  8192 scores in each of 256
// workgroups took 24.3 us from memory, 15 so.
template <int TILES>
__global__ __launch_bounds__(kPickT) void evict_pick_kernel(EvictArgs a) {
    __shared__ int hist[kPickBins];
    __shared__ int tmp[kPickT / 64];
    __shared__ uint32_t range[2];
    __shared__ int found[2];
    constexpr int tile = 4 * kPickT;
    const int tid = threadIdx.x, g = blockIdx.x, b = blockIdx.y;
    const int64_t row = ((int64_t)blockIdx.z * a.batch + b) * a.groups + g;
    const float *x = a.score + row * a.score_stride;
    float *out = a.score_out ? a.score_out + row * a.score_stride : nullptr;
    int32_t *kept = a.kept + row * a.max_budget;
    const EvictSeq s(a, b);
    if (a.len_out && g == 0 && blockIdx.z == 0 && tid == 0) a.len_out[b] = s.n;
    for (int j = s.n + tid; j < a.max_budget; j += kPickT) kept[j] = -1;
    const int from = s.first, to = s.len - s.last;
    const bool held = s.len <= TILES * tile;
    float v[TILES][4];
    auto read = [&](float (&w)[4], int t0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = t0 + 4 * tid + i < s.len ? x[t0 + 4 * tid + i] : 0.f;
    };
#pragma unroll
    for (int k = 0; k < TILES; k++)
        if (held && k * tile < s.len) read(v[k], k * tile);
    // f(the thread's four scores of a tile, their first position), tile by tile
    auto each = [&](auto &&f) __attribute__((always_inline)) {
        if (held) {
#pragma unroll
            for (int k = 0; k < TILES; k++)
                if (k * tile < s.len) f(v[k], k * tile + 4 * tid);
            return;
        }
        for (int t0 = 0; t0 < s.len; t0 += tile) {
            float w[4];
            read(w, t0);
            f(w, t0 + 4 * tid);
        }
    };
    uint32_t limit = 0xffffffffu;  // keys above it stay, and the first `ties` that equal it
    int ties = 0;
    if (s.n < s.len && s.best) {
        if (tid == 0) range[0] = 0xffffffffu, range[1] = 0;
        __syncthreads();
        uint32_t lo = 0xffffffffu, hi = 0;
        each([&](const float (&w)[4], int t) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (t + i >= from && t + i < to) {
                    const uint32_t key = score_key(w[i]);
                    lo = min(lo, key), hi = max(hi, key);
                }
        });
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            lo = min(lo, (uint32_t)__shfl_xor((int)lo, o));
            hi = max(hi, (uint32_t)__shfl_xor((int)hi, o));
        }
        if ((tid & 63) == 0) {
            atomicMin(&range[0], lo);
            atomicMax(&range[1], hi);
        }
        __syncthreads();
        lo = range[0], hi = range[1];
        int need = s.best, bits = hi > lo ? 32 - __builtin_clz(hi - lo) : 0;
        limit = lo, ties = need;  // (all keys equal)
        while (bits) {
            const int shift = max(bits - 11, 0);
            for (int i = tid; i < kPickBins; i += kPickT) hist[i] = 0;
            __syncthreads();
            each([&](const float (&w)[4], int t) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t d = score_key(w[i]) - lo;  // (below lo: past the range too)
                    if (t + i >= from && t + i < to && d >> (bits - 1) < 2) atomicAdd(&hist[d >> shift], 1);
                }
            });
            __syncthreads();
            // two bins a thread, the largest first
            const int top = kPickBins - 1 - 2 * tid, n0 = hist[top], n1 = hist[top - 1];
            int total;
            const int upto = pick_scan(n0 + n1, tmp, total), before = upto - n0 - n1;
            if (before < need && need <= upto) {
                const bool second = before + n0 < need;
                found[0] = second ? top - 1 : top;
                found[1] = second ? before + n0 : before;
            }
            __syncthreads();
            lo += (uint32_t)found[0] << shift;
            need -= found[1];
            limit = lo, ties = need;
            if (hist[found[0]] == need && lo) {  // all of the bin
                limit = lo - 1, ties = 0;
                break;
            }
            bits = shift;
            __syncthreads();
        }
    }
    int kept_n = 0, tie_n = 0;  // kept for certain so far, ties so far
    each([&](const float (&w)[4], int t) __attribute__((always_inline)) {
        int sure = 0, tie = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t key = score_key(w[i]);
            const bool mid = t + i >= from && t + i < to;
            if (t + i < s.len && (s.n == s.len || !mid || key > limit)) sure |= 1 << i;
            else if (mid && key == limit) tie |= 1 << i;
        }
        const int mine = __popc(sure) | __popc(tie) << 16;
        int total;
        const int before = pick_scan(mine, tmp, total) - mine;  // (all of the tile is read)
        int c = kept_n + (before & 0xffff), e = tie_n + (before >> 16);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const bool yes = (sure >> i & 1) || ((tie >> i & 1) && e < ties);
            const int j = c + min(e, ties);
            c += sure >> i & 1, e += tie >> i & 1;
            if (yes && j < s.n) {
                kept[j] = t + i;
                if (out) out[j] = w[i];
            }
        }
        kept_n += total & 0xffff, tie_n += total >> 16;
    });
    if (!out) return;
    __syncthreads();
    for (int t = s.n + tid; t < s.len; t += kPickT) out[t] = 0.f;
}

constexpr int kMoveT = 256, kMoveU = 8;
constexpr int kMoveWgs = 1024;
constexpr int kMovePages = 2048;  // entries of a sequence's table that fit LDS

// Rows of one group of one plane (K or V of a layer), some of its columns.  Row j
// takes position kept[j] >= j, so that rows go down in order: a pass reads its
// rows into registers and stores them when every wave has read; what later
// passes read lies behind what this one writes.  The places of the next pass's rows are
// looked up under this one's loads.  Bound by HBM where there are workgroups enough to
// have their passes (32 KB) cover its latency; columns are cut to 64 bytes for that:
// 8 sequences x 2048 rows x 1 KB in 8 layers took 210 us (2.6 TB/s) with a workgroup a
// group, 115 (4.7 TB/s read and written) with 128 bytes of it.
__global__ __launch_bounds__(kMoveT) void evict_move_kernel(EvictArgs a, int log_c) {
    __shared__ int pages[kMovePages];
    const int tid = threadIdx.x, gb = blockIdx.y, g = gb % a.groups, b = gb / a.groups;
    const int layer = a.one ? blockIdx.z : blockIdx.z >> 1;
    const EvictSeq s(a, b);
    if (s.n >= s.len) return;
    const int32_t *kept = a.kept + (((int64_t)layer * a.batch + b) * a.groups + g) * a.max_budget;
    const int32_t *tab = a.tab ? a.tab + (int64_t)b * a.tab_stride : nullptr;
    const int used = a.tab ? ((s.len - 1) >> a.shift) + 1 : 0;
    const bool in_lds = used <= kMovePages;
    if (in_lds)
        for (int i = tid; i < used; i += kMoveT) pages[i] = tab[i];
    __syncthreads();
    const int c = ((int)blockIdx.x << log_c) + (tid & ((1 << log_c) - 1)), r0 = tid >> log_c, step = kMoveT >> log_c;
    char *base = (!a.one && (blockIdx.z & 1) ? a.v : a.k) + layer * a.layer_b +
                 ((int64_t)g * a.cols + min(c, a.cols - 1)) * 16;
    // byte offset of position t, < 0 where the cache has none
    auto place = [&](int t) __attribute__((always_inline)) -> int64_t {
        if (!a.tab) return b * a.seq_b + t * a.rb;
        const int pg = t >> a.shift, phys = in_lds ? pages[pg] : tab[pg];
        if (phys < 0 || phys >= a.n_pages) return -1;
        return (((int64_t)phys << a.shift) + (t & ((1 << a.shift) - 1))) * a.rb;
    };
    const int rows = step * kMoveU, passes = (s.n + rows - 1) / rows;
    int next[kMoveU];
    auto look = [&](int p) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kMoveU; u++) {
            const int j = p * rows + u * step + r0;
            next[u] = j < s.n ? kept[j] : -1;
        }
    };
    look(0);
    for (int p = 0; p < passes; p++) {  // the same for every wave
        u32x4 x[kMoveU];
        int64_t to[kMoveU];
#pragma unroll
        for (int u = 0; u < kMoveU; u++) {
            const int j = p * rows + u * step + r0, t = next[u];
            to[u] = -1;
            if (t > j && c < a.cols) {
                const int64_t from = place(t);
                if (from >= 0) x[u] = *(const u32x4 *)(base + from), to[u] = place(j);
            }
        }
        look(p + 1);
        // this wave's loads have come, then every wave's
#pragma unroll
        for (int u = 0; u < kMoveU; u++) asm volatile("" : "+v"(x[u])::"memory");
        asm volatile("s_barrier" ::: "memory");
#pragma unroll
        for (int u = 0; u < kMoveU; u++)
            if (to[u] >= 0) *(u32x4 *)(base + to[u]) = x[u];
    }
}

static bool overlap(const void *a, size_t na, const void *b, size_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a && b && na && nb && x < y + nb && y < x + na;
}

static int kv_evict(const char *fn, EvictArgs a, int dtype, int64_t kv_stride, int64_t seq_stride, int kv_dim,
                    int n_layer, int64_t layer_stride, void *stream) {
    if (!dtype_ok(dtype)) return set_error(ULLM_HIP_E_UNSUPPORTED, "%s: dtype %d", fn, dtype);
    if (a.batch < 0 || a.groups < 1 || n_layer < 1 || n_layer > 32767 || (int64_t)a.batch * a.groups > 65535)
        return set_error(ULLM_HIP_E_INVALID, "%s: bad n_layer, or batch * groups not in 0..65535", fn);
    if (kv_dim < 1 || kv_dim % a.groups || kv_stride < kv_dim || seq_stride < 0 || layer_stride < 0)
        return set_error(ULLM_HIP_E_INVALID, "%s: bad kv_dim/strides, or kv_dim no multiple of groups", fn);
    if (a.max_budget < 0 || a.sink < 0 || a.recent < 0 || a.score_stride < 0 || a.score_stride > 1 << 30)
        return set_error(ULLM_HIP_E_INVALID, "%s: max_budget, sink or recent < 0, or score_stride not in 0..2^30", fn);
    // (a grid has less than 2^32 threads)
    if ((int64_t)n_layer * a.batch * a.groups >= 1 << 22 || (int64_t)n_layer * a.batch * kv_dim >= 1ll << 28)
        return set_error(ULLM_HIP_E_INVALID, "%s: too many layers, sequences and groups", fn);
    if ((n_layer > 1 && layer_stride < kv_dim) || (!a.tab && !rows_apart(a.batch, seq_stride, kv_stride, kv_dim)))
        return set_error(ULLM_HIP_E_INVALID, "%s: layers or sequences share rows", fn);
    if (a.batch == 0) return ULLM_HIP_OK;
    const int eb = dtype_bytes(dtype);
    if (!a.k || !a.v || !a.len || !a.budget || (a.score_stride && !a.score) || (a.max_budget && !a.kept))
        return set_error(ULLM_HIP_E_INVALID, "%s: null tensor pointer", fn);
    if (((uintptr_t)a.k | (uintptr_t)a.v) & 15 || (int64_t)kv_dim / a.groups * eb % 16 || kv_stride * eb % 16 ||
        seq_stride * eb % 16 || layer_stride * eb % 16)
        return set_error(ULLM_HIP_E_INVALID, "%s: caches, rows, groups and strides must be 16-byte aligned", fn);
    const size_t rows = (size_t)n_layer * a.batch * a.groups, nb = 4 * (size_t)a.batch;
    const size_t ns = 4 * rows * a.score_stride, nk = 4 * rows * a.max_budget;
    if (overlap(a.len_out, nb, a.len, nb) || overlap(a.len_out, nb, a.budget, nb) || overlap(a.kept, nk, a.len, nb) ||
        overlap(a.kept, nk, a.budget, nb) || overlap(a.kept, nk, a.score, ns) || overlap(a.kept, nk, a.len_out, nb) ||
        overlap(a.len_out, nb, a.score, ns) || overlap(a.kept, nk, a.score_out, ns) ||
        overlap(a.len_out, nb, a.score_out, ns) || overlap(a.score_out, ns, a.len, nb) ||
        overlap(a.score_out, ns, a.budget, nb))
        return set_error(ULLM_HIP_E_INVALID, "%s: an output overlaps an input or another output", fn);
    if (a.tab) {
        const size_t nt = 4 * (size_t)a.batch * a.tab_stride;
        if (overlap(a.tab, nt, a.kept, nk) || overlap(a.tab, nt, a.len_out, nb) || overlap(a.tab, nt, a.score_out, ns))
            return set_error(ULLM_HIP_E_INVALID, "%s: an output overlaps the block table", fn);
    }
    if (a.score_out && a.score_out != a.score && overlap(a.score_out, ns, a.score, ns))
        return set_error(ULLM_HIP_E_INVALID, "%s: scores_out overlaps scores and is not scores", fn);
    a.n_ctx = (int)std::min<int64_t>(a.n_ctx, a.score_stride);
    a.rb = kv_stride * eb, a.seq_b = a.batch > 1 ? seq_stride * eb : 0, a.layer_b = layer_stride * eb;
    a.cols = (int)((int64_t)kv_dim / a.groups * eb / 16);
    a.one = a.k == a.v;
    hipStream_t st = (hipStream_t)stream;
    const dim3 rows_grid(a.groups, a.batch, n_layer), pick(kPickT);
    const int tiles = (a.n_ctx + 4 * kPickT - 1) / (4 * kPickT);
    if (tiles <= 1) launch_kernel(evict_pick_kernel<1>, rows_grid, pick, 0, st, a);
    else if (tiles <= 2) launch_kernel(evict_pick_kernel<2>, rows_grid, pick, 0, st, a);
    else if (tiles <= 4) launch_kernel(evict_pick_kernel<4>, rows_grid, pick, 0, st, a);
    else launch_kernel(evict_pick_kernel<8>, rows_grid, pick, 0, st, a);
    if (int rc = check_hip(hipGetLastError(), "kv_evict launch")) return rc;
    if (a.n_ctx == 0 || a.max_budget == 0) return ULLM_HIP_OK;
    // columns of a workgroup: those of the group, cut down to 64 bytes until there are
    // workgroups for a round of the card
    int log_c = std::min(8, 32 - __builtin_clz(2 * a.cols - 1) - 1);
    const int64_t planes = (int64_t)(a.one ? 1 : 2) * n_layer * a.batch * a.groups;
    while (log_c > 2 && planes * ((a.cols + (1 << log_c) - 1) >> log_c) < kMoveWgs) log_c--;
    launch_kernel(evict_move_kernel, dim3((a.cols + (1 << log_c) - 1) >> log_c, a.batch * a.groups, (a.one ? 1 : 2) * n_layer),
                  dim3(kMoveT), 0, st, a, log_c);
    return check_hip(hipGetLastError(), "kv_evict launch");
}

}  // namespace ullm

using namespace ullm;

extern "C" int ullm_hip_kv_evict(void *k_cache, void *v_cache, int dtype, int64_t kv_stride, int64_t seq_stride,
                                 int n_ctx, int kv_dim, int n_layer, int64_t layer_stride, const float *scores,
                                 float *scores_out, int64_t score_stride, int groups, const int32_t *seq_lens,
                                 const int32_t *budget, int max_budget, int sink, int recent, int32_t *kept,
                                 int32_t *lens_out, int batch, void *stream) {
    if (n_ctx < 0) return set_error(ULLM_HIP_E_INVALID, "kv_evict: n_ctx < 0");
    const EvictArgs a{(char *)k_cache, (char *)v_cache, 0, 0, 0, nullptr, 0, 0, 0, n_ctx, scores, scores_out, score_stride,
                      seq_lens, budget, max_budget, sink, recent, groups, batch, 0, 0, kept, lens_out};
    return kv_evict("kv_evict", a, dtype, kv_stride, seq_stride, kv_dim, n_layer, layer_stride, stream);
}

extern "C" int ullm_hip_kv_evict_paged(void *k_pages, void *v_pages, int dtype, int64_t kv_stride, int page_size,
                                       int n_pages, int kv_dim, int n_layer, int64_t layer_stride,
                                       const int32_t *block_table, int table_stride, const float *scores,
                                       float *scores_out, int64_t score_stride, int groups, const int32_t *seq_lens,
                                       const int32_t *budget, int max_budget, int sink, int recent, int32_t *kept,
                                       int32_t *lens_out, int batch, void *stream) {
    if (page_size < 1 || (page_size & (page_size - 1)))
        return set_error(ULLM_HIP_E_INVALID, "kv_evict_paged: page_size %d must be a power of two", page_size);
    if (n_pages < 1 || table_stride < 1 || (batch > 0 && !block_table))
        return set_error(ULLM_HIP_E_INVALID, "kv_evict_paged: bad n_pages/block_table");
    const int room = (int)std::min<int64_t>((int64_t)table_stride * page_size, INT_MAX);
    const EvictArgs a{(char *)k_pages, (char *)v_pages, 0, 0, 0, block_table, table_stride, __builtin_ctz(page_size),
                      n_pages, room, scores, scores_out, score_stride, seq_lens, budget, max_budget, sink, recent, groups,
                      batch, 0, 0, kept, lens_out};
    return kv_evict("kv_evict_paged", a, dtype, kv_stride, 0, kv_dim, n_layer, layer_stride, stream);
}
