// Entry points of the drafted trees' attention: checks, the cut and the launch
// (tree_attn.hpp has the kernels).
#include <cmath>
#include "tree_attn.hpp"

namespace ullm {

// The cut of a call: as many slots as make one workgroup a CU (two where they pair
// up: 24 sequences of 1K and 35 rows, 8 kv heads, 21.2 us, by one a CU with all its
// LDS 25.3), or one a sequence.  A workgroup holds as many rows as it can, so that K
// and V are read as few times as can be, unless the keys are too few to give every
// second CU a part of `least` blocks (three tiles a key group, below which the merge
// grows by what the parts shrink): then fewer rows, and more workgroups (26 nodes x 6
// heads at 4K, 2 kv heads, with the merge: 256 rows of a workgroup 18 us, 128 16.7, 64
// 15.4, 32 14.8, in parts of two tiles 16.1 and of four 16.3; 4 sequences of 66 rows x
// 256 with a window of 1K, 4 kv heads, without: 128 rows 16.0, 64 17.6, 32 16.8).
struct TreeCut {
    TreeShape shape;
    TreePlan plan;
    int64_t rows;  // of the scratch
};
static TreeCut tree_cut(int dtype, int batch, int nodes, int max_len, int window, int n_head, int n_kv, int D) {
    const int rows = nodes * (n_head / n_kv);
    const int64_t keys = window > 0 ? std::min<int64_t>(max_len, (int64_t)window + nodes) : max_len;
    for (TreeShape s = tree_shape(dtype, D, rows);; s = tree_narrower(dtype, D, s)) {
        TreePlan p{};
        p.batch = batch, p.n_kv = n_kv;
        p.row_tiles = (rows + s.rows() - 1) / s.rows();
        p.least = s.wr == 8 ? 4 : 3 * s.wk;
        const int64_t units = (int64_t)n_kv * p.row_tiles;
        const int64_t most = batch * ((keys / 32 + 2 + p.least - 1) / p.least);
        const bool pairs = tree_pairs(D * dtype_bytes(dtype), s.wr);
        if (s.wr > 1 && most * units < (pairs ? 512 : 128)) continue;
        p.slots = batch;
        if (batch <= 256) p.slots = std::max(batch, (int)std::min<int64_t>((pairs ? 512 : 256) / units, most));
        return {s, p, p.slots > batch ? p.slots * units * s.rows() : 0};
    }
}
static size_t tree_bytes(int64_t rows, int batch, int D) {
    return rows ? (size_t)rows * (D * 4 + 8) + 8 * (size_t)batch + 256 : 0;
}

static int attn_tree(const char *fn, TreeArgs a, TreeKv kv, int dtype, int64_t kv_stride, int batch, int n_kv_head,
                     int head_dim, float scale, int out_dtype, void *ws, size_t ws_bytes, void *stream) {
    if (!dtype_ok(dtype)) return set_error(ULLM_HIP_E_UNSUPPORTED, "%s: dtype %d", fn, dtype);
    if (out_dtype != dtype && out_dtype != ULLM_DT_F32)
        return set_error(ULLM_HIP_E_UNSUPPORTED, "%s: out dtype %d with a cache of dtype %d", fn, out_dtype, dtype);
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return set_error(ULLM_HIP_E_UNSUPPORTED, "%s: head_dim %d not in {64,128,256}", fn, head_dim);
    if (batch < 0 || batch > 65535 || a.nodes < 0 || a.nodes > 1024)
        return set_error(ULLM_HIP_E_INVALID, "%s: batch %d not in 0..65535 or max_nodes %d not in 0..1024", fn, batch,
                         a.nodes);
    if (a.n_head < 1 || n_kv_head < 1 || a.n_head % n_kv_head || a.n_head > 65535)
        return set_error(ULLM_HIP_E_INVALID, "%s: bad heads", fn);
    // (a grid has less than 2^32 threads)
    if ((int64_t)a.nodes * a.n_head > 1 << 23) return set_error(ULLM_HIP_E_INVALID, "%s: too many rows", fn);
    if (a.max_len < 0 || a.window < 0) return set_error(ULLM_HIP_E_INVALID, "%s: bad max_len/window", fn);
    if (kv_stride < (int64_t)n_kv_head * head_dim || kv_stride > 0x7fffffff / 256)
        return set_error(ULLM_HIP_E_INVALID, "%s: kv_stride %lld", fn, (long long)kv_stride);
    if (batch == 0 || a.nodes == 0) return ULLM_HIP_OK;
    if (!a.q || !kv.k || !kv.v || !a.len || !a.out) return set_error(ULLM_HIP_E_INVALID, "%s: null tensor pointer", fn);
    if (a.window > 0 && a.mask && !a.pos)
        return set_error(ULLM_HIP_E_INVALID, "%s: a window over a tree needs its positions", fn);
    const int eb = dtype_bytes(dtype);
    if (((uintptr_t)a.q | (uintptr_t)kv.k | (uintptr_t)kv.v | (uintptr_t)a.out) & 15 || kv_stride * eb % 16 ||
        kv.seq_b % 16)
        return set_error(ULLM_HIP_E_INVALID, "%s: tensors and row strides must be 16-byte aligned", fn);
    a.words = 2 * ((a.nodes + 63) / 64);
    a.kv_mul = a.n_head / n_kv_head;
    a.inv_g = a.kv_mul == 1 ? 0xffffffffu : (uint32_t)((1ull << 32) / a.kv_mul);
    a.neg = scale < 0.f;
    // (a scale of 0 by the least normal number: 0 times a masked score of -inf is none)
    a.qs = std::max(std::fabs(scale) * kLog2e, 1.17549435e-38f);
    kv.rb = kv_stride * eb;
    TreeCut cut = tree_cut(dtype, batch, a.nodes, a.max_len, a.window, a.n_head, n_kv_head, head_dim);
    TreePlan &p = cut.plan;
    if ((int64_t)p.slots * n_kv_head * p.row_tiles > (1 << 23) - 8)
        return set_error(ULLM_HIP_E_INVALID, "%s: too many rows", fn);
    if (const size_t need = tree_bytes(cut.rows, batch, head_dim)) {
        if (!ws || ws_bytes < need || (uintptr_t)ws & 255)
            return set_error(ULLM_HIP_E_WORKSPACE, "%s: workspace of %zu bytes, 256-byte aligned, needed", fn, need);
        p.o = (float *)ws;
        p.ml = (float2 *)(p.o + cut.rows * head_dim);
        p.seq = (int2 *)(p.ml + cut.rows);
    }
    const TreeCall c{cut.shape, a, kv, p, head_dim, out_dtype == ULLM_DT_F32, (hipStream_t)stream};
    if (dtype == ULLM_DT_F32) launch_tree_f32(c);
    else if (dtype == ULLM_DT_F16) launch_tree_f16(c);
    else launch_tree_bf16(c);
    return check_hip(hipGetLastError(), "attn_tree launch");
}

}  // namespace ullm

using namespace ullm;

extern "C" int ullm_hip_attn_tree(const void *q, const void *k_cache, const void *v_cache, int dtype,
                                  int64_t kv_stride, int64_t seq_stride, const int64_t *mask,
                                  const int32_t *seq_lens, const int32_t *n_nodes, const int32_t *positions,
                                  int max_nodes, int max_len, int window, int batch, int n_head, int n_kv_head,
                                  int head_dim, float scale, void *out, int out_dtype, void *workspace,
                                  size_t workspace_bytes, void *stream) {
    if (seq_stride < 0) return set_error(ULLM_HIP_E_INVALID, "attn_tree: seq_stride < 0");
    const TreeArgs a{q, (const uint32_t *)mask, seq_lens, n_nodes, positions, max_nodes, 0, max_len, window, n_head, 1,
                     0, 0.f, 0, out};
    const TreeKv kv{(const char *)k_cache, (const char *)v_cache, 0,
                    batch > 1 && dtype_ok(dtype) ? seq_stride * dtype_bytes(dtype) : 0, nullptr, 0, 0, 0};
    return attn_tree("attn_tree", a, kv, dtype, kv_stride, batch, n_kv_head, head_dim, scale, out_dtype, workspace,
                     workspace_bytes, stream);
}

extern "C" int ullm_hip_attn_tree_paged(const void *q, const void *k_pages, const void *v_pages, int dtype,
                                        int64_t kv_stride, int page_size, int n_pages, const int32_t *block_table,
                                        int table_stride, const int64_t *mask, const int32_t *seq_lens,
                                        const int32_t *n_nodes, const int32_t *positions, int max_nodes, int max_len,
                                        int window, int batch, int n_head, int n_kv_head, int head_dim, float scale,
                                        void *out, int out_dtype, void *workspace, size_t workspace_bytes,
                                        void *stream) {
    if (page_size < 32 || (page_size & (page_size - 1)))
        return set_error(ULLM_HIP_E_INVALID, "attn_tree_paged: page_size %d must be a power of two >= 32", page_size);
    if (n_pages < 1 || table_stride < 1 || (int64_t)table_stride * page_size < max_len)
        return set_error(ULLM_HIP_E_INVALID, "attn_tree_paged: n_pages %d, table of %d pages for max_len %d", n_pages,
                         table_stride, max_len);
    if (batch > 0 && max_nodes > 0 && !block_table)
        return set_error(ULLM_HIP_E_INVALID, "attn_tree_paged: null tensor pointer");
    const TreeArgs a{q, (const uint32_t *)mask, seq_lens, n_nodes, positions, max_nodes, 0, max_len, window, n_head, 1,
                     0, 0.f, 0, out};
    const TreeKv kv{(const char *)k_pages, (const char *)v_pages, 0, 0, block_table, table_stride,
                    __builtin_ctz(page_size), n_pages};
    return attn_tree("attn_tree_paged", a, kv, dtype, kv_stride, batch, n_kv_head, head_dim, scale, out_dtype,
                     workspace, workspace_bytes, stream);
}

extern "C" size_t ullm_hip_tree_workspace_bytes(int dtype, int batch, int max_nodes, int max_len, int window,
                                                int n_head, int n_kv_head, int head_dim) {
    if (!dtype_ok(dtype) || (head_dim != 64 && head_dim != 128 && head_dim != 256) || batch < 1 || max_nodes < 1 ||
        max_nodes > 1024 || n_head < 1 || n_kv_head < 1 || n_head % n_kv_head || n_head > 65535 || max_len < 0 ||
        (int64_t)max_nodes * n_head > 1 << 23)
        return 0;
    // For every call with fewer sequences, nodes and positions too: at most 256 cut
    // sequences, and 256 workgroups of eight waves or 512 of fewer, of the widest
    // shape's rows (of eight waves': or 512 of half), where there are keys to cut.
    const int64_t keys = window > 0 ? std::min<int64_t>(max_len, (int64_t)window + max_nodes) : max_len;
    const TreeShape s = tree_shape(dtype, head_dim, max_nodes * (n_head / n_kv_head));
    return keys / 32 + 2 > 2 ? tree_bytes((s.wr == 8 ? 256 : 512) * (int64_t)s.rows(), 256, head_dim) : 0;
}
