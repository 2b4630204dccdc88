// Rows and pages of a KV cache moved, shared, copied and given back:
// ullm_hip_kv_accept(_paged) and ullm_hip_kv_pages_update.
#include <algorithm>
#include <climits>
#include "common.hpp"
#include "wave.hpp"

namespace ullm {

// ---- the accepted rows of a drafted tree ----
// Row len + j of sequence b takes what row len + path[b][j] held, j < count[b],
// for K and V of every layer (2 n_layer planes, n_layer where V is K).  A workgroup takes a sequence
// and some planes: it finds its rows' places once, then for 2^log_c columns of
// 16 bytes at a time reads all source rows into registers and stores after a
// barrier, the next columns' loads in flight.  So any path is right, also one
// that is not increasing or names a row twice, and no other workgroup touches
// those columns.  Bound by HBM: 32 sequences x 11 moved rows of 2 KB in 36
// layers (104 MB) take 20.3 us (5.1 TB/s); 61.9 with a workgroup per 512-byte
// slice of one plane, which finds its rows' places anew.
struct AcceptArgs {
    char *k, *v;
    int64_t rb, seq_b, layer_b;  // bytes of a row, from sequence to sequence, from layer to layer
    const int32_t *tab;          // null: contiguous, n_ctx rows
    int tab_stride, shift, n_pages, n_ctx;
    const int32_t *path, *count, *len;
    int path_stride, cols;  // 16-byte columns of a row that are moved
    int one;                // K and V are the same memory, which moves once
    int32_t *len_out;
};
constexpr int kAcceptT = 256, kAcceptU = 8;
constexpr int kAcceptMax = 1024;  // nodes of a path
constexpr int kAcceptWgs = 1024;  // workgroups aimed at: four a CU

// Byte offset of position t of sequence b, < 0 where the cache has none.
__device__ __forceinline__ int64_t accept_row(const AcceptArgs &a, int b, int64_t t) {
    if (t < 0) return -1;
    if (!a.tab) return t < a.n_ctx ? b * a.seq_b + t * a.rb : -1;
    const int64_t pg = t >> a.shift;
    const int phys = pg < a.tab_stride ? a.tab[(int64_t)b * a.tab_stride + pg] : -1;
    if (phys < 0 || phys >= a.n_pages) return -1;
    return (((int64_t)phys << a.shift) + (t & ((1 << a.shift) - 1))) * a.rb;
}

// The planes' rows in passes of kAcceptT * U pieces of 16 bytes.
template <int U>
__device__ __forceinline__ void accept_planes(const AcceptArgs &a, const int64_t *sfrom, const int64_t *sto, int n,
                                              int log_c, int p0, int p1) {
    const int tid = threadIdx.x, c = tid & ((1 << log_c) - 1), r0 = tid >> log_c, step = kAcceptT >> log_c;
    int64_t from[U], to[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int j = r0 + u * step;
        from[u] = j < n ? sfrom[j] : 0;  // (what is not moved reads row 0 of the plane)
        to[u] = j < n ? sto[j] : -1;
    }
    const int gx = gridDim.x, passes = (((a.cols - 1) >> log_c) - (int)blockIdx.x + gx) / gx;
    auto col = [&](int i) { return (((int)blockIdx.x + i % passes * gx) << log_c) + c; };
    auto base = [&](int i) {  // of pass i over this workgroup's planes and columns
        const int p = p0 + i / passes, layer = a.one ? p : p >> 1;
        return (!a.one && (p & 1) ? a.v : a.k) + layer * a.layer_b;
    };
    auto load = [&](int i, u32x4 (&x)[U]) {
        const char *at = base(i) + (int64_t)min(col(i), a.cols - 1) * 16;
#pragma unroll
        for (int u = 0; u < U; u++) x[u] = *(const u32x4 *)(at + from[u]);
    };
    auto store = [&](int i, u32x4 (&x)[U]) {
        // this wave's loads have come, then every wave's
#pragma unroll
        for (int u = 0; u < U; u++) asm volatile("" : "+v"(x[u])::"memory");
        asm volatile("s_barrier" ::: "memory");
        char *at = base(i) + (int64_t)col(i) * 16;
        if (col(i) < a.cols)
#pragma unroll
            for (int u = 0; u < U; u++)
                if (to[u] >= 0) *(u32x4 *)(at + to[u]) = x[u];
    };
    const int total = (p1 - p0) * passes;  // the same for every wave
    u32x4 x[U], y[U];
    if (total <= 0) return;
    load(0, x);
    for (int i = 0; i < total; i += 2) {
        load(min(i + 1, total - 1), y);
        store(i, x);
        if (i + 1 >= total) break;
        load(min(i + 2, total - 1), x);
        store(i + 1, y);
    }
}

__global__ __launch_bounds__(kAcceptT) void kv_accept_kernel(AcceptArgs a, int planes, int per) {
    __shared__ int64_t sfrom[kAcceptMax], sto[kAcceptMax];
    const int tid = threadIdx.x, b = blockIdx.y;
    const int len = a.len[b], n = min(max(a.count[b], 0), a.path_stride);
    if (a.len_out && blockIdx.x == 0 && blockIdx.z == 0 && tid == 0) a.len_out[b] = len + n;
    for (int j = tid; j < n; j += kAcceptT) {
        const int node = a.path[(int64_t)b * a.path_stride + j];
        int64_t from = 0, to = -1;
        if (node >= 0 && node != j) {
            from = accept_row(a, b, (int64_t)len + node);
            to = accept_row(a, b, (int64_t)len + j);
            if (from < 0) from = 0, to = -1;
        }
        sfrom[j] = from;
        sto[j] = to;
    }
    if (n == 0) return;
    __syncthreads();
    // columns of a pass: as many as kAcceptU pieces of every thread cover for n rows
    int log_c = 31 - __builtin_clz(kAcceptT * kAcceptU / n);
    while (log_c > 0 && ((1 << log_c) > kAcceptT || (1 << (log_c - 1)) >= a.cols)) log_c--;
    const int p0 = (int)blockIdx.z * per, p1 = min(p0 + per, planes);
    const int pieces = (n + (kAcceptT >> log_c) - 1) / (kAcceptT >> log_c);  // of a thread
    if (pieces <= 1) accept_planes<1>(a, sfrom, sto, n, log_c, p0, p1);
    else if (pieces <= 2) accept_planes<2>(a, sfrom, sto, n, log_c, p0, p1);
    else if (pieces <= 4) accept_planes<4>(a, sfrom, sto, n, log_c, p0, p1);
    else accept_planes<8>(a, sfrom, sto, n, log_c, p0, p1);
}

static bool overlap(const void *a, size_t na, const void *b, size_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a && b && x < y + nb && y < x + na;
}

static int kv_accept(const char *fn, AcceptArgs a, int dtype, int64_t kv_stride, int64_t seq_stride, int kv_dim,
                     int n_layer, int64_t layer_stride, int batch, void *stream) {
    if (!dtype_ok(dtype)) return set_error(ULLM_HIP_E_UNSUPPORTED, "%s: dtype %d", fn, dtype);
    if (batch < 0 || batch > 65535 || a.path_stride < 0 || a.path_stride > kAcceptMax)
        return set_error(ULLM_HIP_E_INVALID, "%s: batch %d not in 0..65535 or path of %d not in 0..%d", fn, batch,
                         a.path_stride, kAcceptMax);
    if (n_layer < 1 || n_layer > 32767 || kv_dim < 1 || kv_stride < kv_dim || seq_stride < 0 || layer_stride < 0)
        return set_error(ULLM_HIP_E_INVALID, "%s: bad n_layer/kv_dim/strides", fn);
    if ((n_layer > 1 && layer_stride < kv_dim) || (!a.tab && !rows_apart(batch, seq_stride, kv_stride, kv_dim)))
        return set_error(ULLM_HIP_E_INVALID, "%s: layers or sequences share rows", fn);
    if (batch == 0) return ULLM_HIP_OK;
    const int eb = dtype_bytes(dtype);
    if (!a.k || !a.v || !a.count || !a.len || (!a.path && a.path_stride))
        return set_error(ULLM_HIP_E_INVALID, "%s: null tensor pointer", fn);
    if (((uintptr_t)a.k | (uintptr_t)a.v) & 15 || (int64_t)kv_dim * eb % 16 || kv_stride * eb % 16 ||
        seq_stride * eb % 16 || layer_stride * eb % 16)
        return set_error(ULLM_HIP_E_INVALID, "%s: caches, rows and strides must be 16-byte aligned", fn);
    // (one workgroup of a sequence writes its length while the others still read)
    const size_t nl = 4 * (size_t)batch;
    if (overlap(a.len_out, nl, a.len, nl) || overlap(a.len_out, nl, a.count, nl) ||
        overlap(a.len_out, nl, a.path, nl * a.path_stride) || overlap(a.len_out, nl, a.tab, nl * a.tab_stride))
        return set_error(ULLM_HIP_E_INVALID, "%s: lens_out overlaps seq_lens, n_accept, path or block_table", fn);
    a.rb = kv_stride * eb, a.seq_b = batch > 1 ? seq_stride * eb : 0, a.layer_b = layer_stride * eb;
    a.cols = (int)((int64_t)kv_dim * eb / 16);
    a.one = a.k == a.v;
    const int planes = a.tab || a.n_ctx ? (a.one ? 1 : 2) * n_layer : 0;  // (no rows: only the lengths)
    const int gx = std::max(1, std::min((a.cols + 255) / 256, kAcceptWgs / batch));  // passes of 256 columns side by side
    const int64_t wgs = (int64_t)batch * gx * planes;
    const int per = (int)std::max<int64_t>(1, std::min<int64_t>(planes, wgs / kAcceptWgs));
    launch_kernel(kv_accept_kernel, dim3(gx, batch, std::max(1, (planes + per - 1) / per)), dim3(kAcceptT), 0, (hipStream_t)stream, a,
                  planes, per);
    return check_hip(hipGetLastError(), "kv_accept launch");
}

// ---- the block table of the next step ----
// Sequence s of the new table goes on from sequence parent[s] of the old one
// (none: starts empty), keeps min(its length, capacity[s]) positions and has
// pages for capacity[s].  Pages that kept positions fill are shared; a page
// that they fill in part is the first such sequence's own, if it is no one's
// whole page and not held, and copied for every other.  New pages are those
// that nothing keeps, lowest number first.
struct PagesArgs {
    char *k, *v;
    int64_t rb, layer_b;  // bytes of a row, from layer to layer
    int cols;             // 16-byte columns of a row that are copied; 0: whole rows
    const int32_t *tab, *len, *parent, *cap;
    const uint8_t *held;
    int32_t *tab_out, *len_out, *info;
    int stride, n_seq, out_stride, n_out, n_pages, shift;
    // workspace
    int32_t *owner, *free_list, *total;  // [n_pages], [n_pages], [2]: pages free, pages asked for
    struct PagesSeq *seq;
};
// What becomes of one sequence: old row, whole kept pages, kept positions of
// the next one, pages needed, the first of its new ones, and the part-filled
// page (-1: none) with whether it is kept as it is.
struct PagesSeq {
    int32_t p, full, part, need, first, last, keeps, pad;
};
constexpr int kPagesT = 1024, kPagesU = 8;
constexpr int kPagesMax = 1 << 20;  // pages of a pool: a bit each in LDS

// Exclusive sum of v over the workgroup, and the total.
__device__ __forceinline__ int block_scan(int v, int *tmp, int &total) {
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int x = wave_scan(v);
    __syncthreads();
    if (lane == 63) tmp[w] = x;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kPagesT / 64; i++) {
        if (i < w) before += tmp[i];
        total += tmp[i];
    }
    return before + x - v;
}

// One workgroup: marks the pages that stay in a bitmap in LDS, settles the
// part-filled ones, and lists the free ones in order.  Bound by the latency of its
// dependent loads (parent, length, table entry, page), which is why a thread keeps
// the first sequence that is its own in registers and every loop has its loads in
// flight together: 64 sequences of up to 16K in pages of 32 took 23.3 us with a
// load at a time, 12.7 with 8 and the sequences kept in memory, 11.4 so.
__global__ __launch_bounds__(kPagesT) void pages_plan_kernel(PagesArgs a) {
    extern __shared__ uint32_t bits[];  // pages that stay: held or kept
    __shared__ int tmp[kPagesT / 64];
    __shared__ int2 rows[kPagesT];  // old row and whole kept pages of the first sequences
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int words = (a.n_pages + 31) / 32;
    const int64_t room = (int64_t)a.out_stride << a.shift, had = (int64_t)a.stride << a.shift;
    auto first_look = [&](int s) {
        const int p = a.parent[s], cap = (int)min((int64_t)max(a.cap[s], 0), room);
        const int kept = p >= 0 && p < a.n_seq ? (int)min(min((int64_t)max(a.len[p], 0), had), (int64_t)cap) : 0;
        const int full = kept >> a.shift, part = kept & ((1 << a.shift) - 1);
        int last = part ? a.tab[(int64_t)p * a.stride + full] : -1;
        if (last < 0 || last >= a.n_pages) last = -1;
        if (last >= 0) __hip_atomic_store(a.owner + last, INT_MAX, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        return PagesSeq{p, full, part, (int)((cap + (1ll << a.shift) - 1) >> a.shift), 0, last, 0, 0};
    };
    PagesSeq mine{};  // of sequence tid
    if (tid < a.n_out) {
        mine = first_look(tid);
        rows[tid] = int2{mine.p, mine.full};
    }
    for (int s = tid + kPagesT; s < a.n_out; s += kPagesT) a.seq[s] = first_look(s);
    if (a.held) {  // 64 pages a load of a wave
        for (int c0 = wave; c0 * 64 < a.n_pages; c0 += kPagesU * (kPagesT / 64)) {
            bool held[kPagesU];
#pragma unroll
            for (int u = 0; u < kPagesU; u++) {
                const int pg = (c0 + u * (kPagesT / 64)) * 64 + lane;
                held[u] = pg < a.n_pages && a.held[pg];
            }
#pragma unroll
            for (int u = 0; u < kPagesU; u++) {
                const int c = c0 + u * (kPagesT / 64);
                const uint64_t m = __ballot(held[u]);
                if (lane < 2 && 2 * c + lane < words) bits[2 * c + lane] = (uint32_t)(m >> (32 * lane));
            }
        }
    } else {
        for (int w = tid; w < words; w += kPagesT) bits[w] = 0;
    }
    __syncthreads();
    if (mine.last >= 0 && tid < a.n_out) atomicMin(a.owner + mine.last, tid);
    for (int s = tid + kPagesT; s < a.n_out; s += kPagesT)
        if (a.seq[s].last >= 0) atomicMin(a.owner + a.seq[s].last, s);
    // whole pages: a wave takes a sequence, kPagesU loads of 64 entries in flight
    for (int s = wave; s < a.n_out; s += kPagesT / 64) {
        int2 q = s < kPagesT ? rows[s] : int2{a.seq[s].p, a.seq[s].full};
        const int32_t *row = a.tab + (int64_t)q.x * a.stride;
        for (int j0 = 0; j0 < q.y; j0 += 64 * kPagesU) {
            int pg[kPagesU];
#pragma unroll
            for (int u = 0; u < kPagesU; u++) pg[u] = j0 + u * 64 + lane < q.y ? row[j0 + u * 64 + lane] : -1;
#pragma unroll
            for (int u = 0; u < kPagesU; u++)
                if (pg[u] >= 0 && pg[u] < a.n_pages) atomicOr(&bits[pg[u] >> 5], 1u << (pg[u] & 31));
        }
    }
    __syncthreads();
    // who keeps its part-filled page, and the new pages of each
    auto keeps = [&](const PagesSeq &q, int s) {
        return q.last >= 0 && !(bits[q.last >> 5] >> (q.last & 31) & 1) &&
               __hip_atomic_load(a.owner + q.last, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == s;
    };
    int asked = 0;
    for (int s0 = 0; s0 < a.n_out; s0 += kPagesT) {
        const int s = s0 + tid;
        PagesSeq q = mine;
        int take = 0;
        if (s < a.n_out) {
            if (s0) q = a.seq[s];
            q.keeps = keeps(q, s);
            take = q.need - q.full - q.keeps;
        }
        int total;
        q.first = asked + block_scan(take, tmp, total);
        if (s0 == 0) mine = q;
        if (s < a.n_out) a.seq[s] = q;
        asked += total;
    }
    // (every sum above is behind barriers: all have looked at the marks)
    if (tid < a.n_out && mine.last >= 0) atomicOr(&bits[mine.last >> 5], 1u << (mine.last & 31));
    for (int s = tid + kPagesT; s < a.n_out; s += kPagesT) {
        const int last = a.seq[s].last;
        if (last >= 0) atomicOr(&bits[last >> 5], 1u << (last & 31));
    }
    __syncthreads();
    // the free pages in order, as many as are asked for
    const int per = (words + kPagesT - 1) / kPagesT, w0 = tid * per, w1 = min(w0 + per, words);
    auto free_of = [&](int w) {
        const uint32_t there = w * 32 + 32 <= a.n_pages ? ~0u : (1u << (a.n_pages & 31)) - 1;
        return ~bits[w] & there;
    };
    int count = 0, n_free;
    for (int w = w0; w < w1; w++) count += __popc(free_of(w));
    int rank = block_scan(count, tmp, n_free);
    for (int w = w0; w < w1 && rank < asked; w++)
        for (uint32_t f = free_of(w); f && rank < asked; f &= f - 1) a.free_list[rank++] = w * 32 + __builtin_ctz(f);
    // the new lengths: a part-filled page that should have been copied and could not is lost
    int copies = 0;
    for (int s = tid; s < a.n_out; s += kPagesT) {
        const PagesSeq q = s == tid ? mine : a.seq[s];
        const bool copy = q.last >= 0 && !q.keeps, lost = copy && q.first >= n_free;
        copies += copy && !lost;
        a.len_out[s] = (q.full << a.shift) + (lost ? 0 : q.part);
    }
    int n_copies;
    block_scan(copies, tmp, n_copies);
    if (tid == 0) {
        a.total[0] = n_free;
        a.info[0] = n_copies;
        a.info[1] = min(asked, n_free);
        a.info[2] = max(asked - n_free, 0);
    }
}

// Rows of the new table (blockIdx.z == 0), and the copies of part-filled pages
// in K and V of every layer.
__global__ __launch_bounds__(256) void pages_apply_kernel(PagesArgs a) {
    const int s = blockIdx.y, tid = threadIdx.x, n_free = a.total[0];
    const PagesSeq q = a.seq[s];
    if (blockIdx.z == 0) {
        for (int j = blockIdx.x * 256 + tid; j < a.out_stride; j += gridDim.x * 256) {
            int pg = -1;
            if (j < q.full) {
                pg = a.tab[(int64_t)q.p * a.stride + j];
                if (pg < 0 || pg >= a.n_pages) pg = -1;
            } else if (j == q.full && q.keeps) {
                pg = q.last;
            } else if (j < q.need) {
                const int nth = q.first + j - q.full - q.keeps;
                if (nth < n_free) pg = a.free_list[nth];
            }
            a.tab_out[(int64_t)s * a.out_stride + j] = pg;
        }
        return;
    }
    if (q.last < 0 || q.keeps || q.first >= n_free) return;
    const int z = blockIdx.z - 1;
    char *base = ((z & 1) ? a.v : a.k) + (z >> 1) * a.layer_b;
    const char *src = base + ((int64_t)q.last << a.shift) * a.rb;
    char *dst = base + ((int64_t)a.free_list[q.first] << a.shift) * a.rb;
    if (!a.cols) {
        const int64_t n16 = q.part * a.rb / 16;
        for (int64_t i = blockIdx.x * 256 + tid; i < n16; i += gridDim.x * 256)
            *(u32x4 *)(dst + i * 16) = *(const u32x4 *)(src + i * 16);
        return;
    }
    // rows of a wider buffer, 2^log_c columns side by side
    const int log_c = a.cols >= 256 ? 8 : 31 - __builtin_clz(2 * a.cols - 1);
    for (int64_t r = blockIdx.x * (256 >> log_c) + (tid >> log_c); r < q.part; r += gridDim.x * (256 >> log_c))
        for (int c = tid & ((1 << log_c) - 1); c < a.cols; c += 1 << log_c)
            *(u32x4 *)(dst + r * a.rb + c * 16ll) = *(const u32x4 *)(src + r * a.rb + c * 16ll);
}

static size_t pages_ws(int n_out, int n_pages) {
    return 256 + (size_t)n_out * sizeof(PagesSeq) + 8 * (size_t)n_pages;
}

}  // namespace ullm

using namespace ullm;

extern "C" int ullm_hip_kv_accept(void *k_cache, void *v_cache, int dtype, int64_t kv_stride, int64_t seq_stride,
                                  int n_ctx, int kv_dim, int n_layer, int64_t layer_stride, const int32_t *path,
                                  int path_stride, const int32_t *n_accept, const int32_t *seq_lens,
                                  int32_t *lens_out, int batch, void *stream) {
    if (n_ctx < 0) return set_error(ULLM_HIP_E_INVALID, "kv_accept: n_ctx < 0");
    const AcceptArgs a{(char *)k_cache, (char *)v_cache, 0, 0, 0, nullptr, 0, 0, 0, n_ctx,
                       path, n_accept, seq_lens, path_stride, 0, 0, lens_out};
    return kv_accept("kv_accept", a, dtype, kv_stride, seq_stride, kv_dim, n_layer, layer_stride, batch, stream);
}

extern "C" int ullm_hip_kv_accept_paged(void *k_pages, void *v_pages, int dtype, int64_t kv_stride, int page_size,
                                        int n_pages, int kv_dim, int n_layer, int64_t layer_stride,
                                        const int32_t *block_table, int table_stride, const int32_t *path,
                                        int path_stride, const int32_t *n_accept, const int32_t *seq_lens,
                                        int32_t *lens_out, int batch, void *stream) {
    if (page_size < 1 || (page_size & (page_size - 1)))
        return set_error(ULLM_HIP_E_INVALID, "kv_accept_paged: page_size %d must be a power of two", page_size);
    if (n_pages < 1 || table_stride < 1 || (batch > 0 && !block_table))
        return set_error(ULLM_HIP_E_INVALID, "kv_accept_paged: bad n_pages/block_table");
    const AcceptArgs a{(char *)k_pages, (char *)v_pages, 0, 0, 0, block_table, table_stride, __builtin_ctz(page_size),
                       n_pages, 0, path, n_accept, seq_lens, path_stride, 0, 0, lens_out};
    return kv_accept("kv_accept_paged", a, dtype, kv_stride, 0, kv_dim, n_layer, layer_stride, batch, stream);
}

extern "C" size_t ullm_hip_kv_pages_workspace_bytes(int n_out, int n_pages) {
    return n_out < 1 || n_pages < 1 ? 0 : pages_ws(n_out, n_pages);
}

// kv_dim 0: whole rows.
static int pages_update(const char *fn, void *k_pages, void *v_pages, int dtype, int64_t kv_stride, int page_size,
                        int n_pages, int kv_dim, int n_layer, int64_t layer_stride, const int32_t *block_table,
                        int table_stride, const int32_t *seq_lens, int n_seq, const int32_t *parent,
                        const int32_t *capacity, const uint8_t *held, int32_t *table_out, int out_stride,
                        int32_t *lens_out, int n_out, int32_t *info, void *workspace, size_t workspace_bytes,
                        void *stream) {
    if (!dtype_ok(dtype)) return set_error(ULLM_HIP_E_UNSUPPORTED, "%s: dtype %d", fn, dtype);
    if (page_size < 1 || (page_size & (page_size - 1)))
        return set_error(ULLM_HIP_E_INVALID, "%s: page_size %d must be a power of two", fn, page_size);
    if (n_pages < 1 || n_pages > kPagesMax)
        return set_error(ULLM_HIP_E_UNSUPPORTED, "%s: n_pages %d not in 1..%d", fn, n_pages, kPagesMax);
    if (n_seq < 0 || n_out < 0 || n_out > 65535 || table_stride < 1 || out_stride < 1 || n_layer < 0 ||
        n_layer > 32767 || kv_stride < 1 || layer_stride < 0)
        return set_error(ULLM_HIP_E_INVALID, "%s: bad sizes", fn);
    if ((int64_t)page_size * table_stride > INT_MAX || (int64_t)page_size * out_stride > INT_MAX)
        return set_error(ULLM_HIP_E_INVALID, "%s: a table of 2^31 positions or more", fn);
    if ((int64_t)n_out * out_stride > INT_MAX)  // (the pages asked for are counted in 32 bits)
        return set_error(ULLM_HIP_E_INVALID, "%s: a table of 2^31 entries or more", fn);
    if (kv_stride < kv_dim || (n_layer > 1 && layer_stride < kv_dim))
        return set_error(ULLM_HIP_E_INVALID, "%s: rows or layers share memory", fn);
    if (n_out == 0) return ULLM_HIP_OK;
    if ((n_layer && (!k_pages || !v_pages)) || (n_seq && (!block_table || !seq_lens)) || !parent || !capacity ||
        !table_out || !lens_out || !info)
        return set_error(ULLM_HIP_E_INVALID, "%s: null tensor pointer", fn);
    const int eb = dtype_bytes(dtype);
    if (((uintptr_t)k_pages | (uintptr_t)v_pages) & 15 || kv_stride * eb % 16 || layer_stride * eb % 16 ||
        (int64_t)kv_dim * eb % 16)
        return set_error(ULLM_HIP_E_INVALID, "%s: pools, rows and strides must be 16-byte aligned", fn);
    const size_t nt = 4 * (size_t)n_out * out_stride, ot = 4 * (size_t)n_seq * table_stride;
    if (overlap(table_out, nt, block_table, ot) || overlap(lens_out, 4 * (size_t)n_out, block_table, ot) ||
        overlap(info, 12, block_table, ot))
        return set_error(ULLM_HIP_E_INVALID, "%s: an output overlaps the old table", fn);
    if (overlap(table_out, nt, lens_out, 4 * (size_t)n_out) || overlap(table_out, nt, info, 12) ||
        overlap(lens_out, 4 * (size_t)n_out, info, 12))
        return set_error(ULLM_HIP_E_INVALID, "%s: the outputs overlap", fn);
    const size_t need = pages_ws(n_out, n_pages);
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace & 255)
        return set_error(ULLM_HIP_E_WORKSPACE, "%s: workspace of %zu bytes, 256-byte aligned, needed", fn, need);
    char *ws = (char *)workspace;
    PagesArgs a{(char *)k_pages, (char *)v_pages, kv_stride * eb, layer_stride * eb,
                kv_dim < kv_stride ? (int)((int64_t)kv_dim * eb / 16) : 0, block_table, seq_lens, parent, capacity,
                held, table_out, lens_out, info, table_stride, n_seq, out_stride, n_out, n_pages,
                __builtin_ctz(page_size), nullptr, nullptr, (int32_t *)ws, (PagesSeq *)(ws + 256)};
    a.owner = (int32_t *)(ws + 256 + (size_t)n_out * sizeof(PagesSeq));
    a.free_list = a.owner + n_pages;
    hipStream_t st = (hipStream_t)stream;
    launch_kernel(pages_plan_kernel, dim3(1), dim3(kPagesT), (size_t)(n_pages + 31) / 32 * 4, st, a);
    if (int rc = check_hip(hipGetLastError(), "kv_pages_update launch")) return rc;
    launch_kernel(pages_apply_kernel, dim3(8, n_out, 1 + 2 * n_layer), dim3(256), 0, st, a);
    return check_hip(hipGetLastError(), "kv_pages_update launch");
}

extern "C" int ullm_hip_kv_pages_update(void *k_pages, void *v_pages, int dtype, int64_t kv_stride, int page_size,
                                        int n_pages, int n_layer, int64_t layer_stride, const int32_t *block_table,
                                        int table_stride, const int32_t *seq_lens, int n_seq, const int32_t *parent,
                                        const int32_t *capacity, const uint8_t *held, int32_t *table_out,
                                        int out_stride, int32_t *lens_out, int n_out, int32_t *info, void *workspace,
                                        size_t workspace_bytes, void *stream) {
    return pages_update("kv_pages_update", k_pages, v_pages, dtype, kv_stride, page_size, n_pages, 0, n_layer,
                        layer_stride, block_table, table_stride, seq_lens, n_seq, parent, capacity, held, table_out,
                        out_stride, lens_out, n_out, info, workspace, workspace_bytes, stream);
}

extern "C" int ullm_hip_kv_pages_update_rows(void *k_pages, void *v_pages, int dtype, int64_t kv_stride,
                                             int page_size, int n_pages, int kv_dim, int n_layer,
                                             int64_t layer_stride, const int32_t *block_table, int table_stride,
                                             const int32_t *seq_lens, int n_seq, const int32_t *parent,
                                             const int32_t *capacity, const uint8_t *held, int32_t *table_out,
                                             int out_stride, int32_t *lens_out, int n_out, int32_t *info,
                                             void *workspace, size_t workspace_bytes, void *stream) {
    if (kv_dim < 1) return set_error(ULLM_HIP_E_INVALID, "kv_pages_update_rows: kv_dim < 1");
    return pages_update("kv_pages_update_rows", k_pages, v_pages, dtype, kv_stride, page_size, n_pages, kv_dim,
                        n_layer, layer_stride, block_table, table_stride, seq_lens, n_seq, parent, capacity, held,
                        table_out, out_stride, lens_out, n_out, info, workspace, workspace_bytes, stream);
}
