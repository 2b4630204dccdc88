// Entry points of the drafted trees' attention: checks, the cut and the launch
// (tree_attn.hpp has the kernels).
#include <cmath>
#include "tree_attn.hpp"

namespace ullm {

// The cut of a call: the shape of a workgroup and the slots along the keys with the
// least estimate, of all shapes that hold the rows and of the sequences whole, in 2, 3,
// 4, 6, .. parts each, or in as many as the card holds workgroups (two a CU where they
// pair up).  Wide workgroups read K and V the fewest times; narrow ones are more and
// start sooner; parts cost the merge and the joined partials.  Measured, us: 4 sequences
// of 64 nodes, 32/4 heads x 128, bf16, 300 tokens 12.6 (16 rows; 256 rows 25.8), 1000 23.3
// (16 rows 22.7, 256 rows 34.2), 4000 43.8 (64 rows 42.3, 256 rows 43.8, 16 rows 63.8); 26
// nodes at 300 tokens, 12/2 heads, 9.9 (256 rows 16.8), at 4000 13.0 (16 rows, in parts; 256
// rows 16.5); 2 sequences of 64 nodes, 32/8 x 128, f32, 4000 tokens 57.7 (128 rows; 64 rows 82).
// Over 69 calls, 65 of them of 16 bits, 300 to 32000 tokens, the choice takes at most 1.14 times the
// best shape's time, but for two (1.17 and 1.23).
struct TreeCut {
    TreeShape shape;
    TreePlan plan;
    int64_t rows;  // of the scratch
};
// Microseconds that a workgroup of 16, 32, 64, 128 or 256 rows takes for 32 keys, where
// there are few of them and where they fill the card (8 kv heads, 8 and 64 sequences of
// 416 and 1440 tokens, uncut).
struct TreeCost {
    float few, full;
};
static constexpr TreeCost kTreeCost[2][3][5] = {
    {{{.32f, .60f}, {.50f, .57f}, {.40f, .62f}, {.73f, 1.11f}, {.88f, .95f}},       // 16 bits x 64
     {{.46f, 1.56f}, {.75f, 1.58f}, {.62f, 1.67f}, {1.01f, 2.10f}, {1.17f, 1.34f}},  // x 128
     {{1.18f, 2.88f}, {1.19f, 3.05f}, {1.06f, 3.17f}, {1.17f, 1.96f}, {}}},          // x 256
    {{{.60f, 1.55f}, {.70f, 1.78f}, {1.28f, 2.63f}, {2.11f, 3.51f}, {2.29f, 2.59f}},  // f32 x 64
     {{1.50f, 3.01f}, {1.44f, 3.36f}, {2.35f, 4.90f}, {2.55f, 3.35f}, {}},
     {{2.71f, 3.44f}, {2.80f, 3.72f}, {4.55f, 5.31f}, {7.68f, 7.58f}, {}}}};
static TreeCut tree_cut(int dtype, int batch, int nodes, int max_len, int window, int n_head, int n_kv, int D) {
    const int rows = nodes * (n_head / n_kv), rb = D * dtype_bytes(dtype);
    const int64_t keys = window > 0 ? std::min<int64_t>(max_len, (int64_t)window + nodes) : max_len;
    const int64_t blocks = keys / 32 + 1;
    TreeCut best{};
    float least = INFINITY;
    for (TreeShape s = tree_shape(dtype, D, rows);; s = tree_narrower(dtype, D, s)) {
        const int row_tiles = (rows + s.rows() - 1) / s.rows();
        const int64_t units = (int64_t)n_kv * row_tiles, room = tree_pairs(rb, s.wr) ? 512 : 256;
        TreeCost c = kTreeCost[dtype == ULLM_DT_F32][D / 128][__builtin_ctz(s.rows()) - 4];
        // Up to 192 of 256 rows a SIMD's two waves hold three row tiles, not four (16 bits x
        // 128, 192 rows: .94 and 1.15 a block; f32 x 64 1.93 and 2.04).
        if (s.rows() == 256 && rows <= 192) c.few *= .8f, c.full *= .8f;
        const int part = s.wr == 8 ? 4 : 2 * s.wk;  // blocks that a part has at least
        // Where they fill the card they wait for memory or for the matrix units: of what they
        // read row tiles of one kv head share a part, but never less than the products take.
        // (It is memory that they wait for where `full` is within .9 and 1.25 of the reads of
        // K and V at 5.3 TB/s.  The part that tiles share goes by the square root of their
        // number: the number itself chose too narrow shapes.  The products of a row are put at
        // a third over the widest 16-bit shape's time of one, which they bind, and over f32 at
        // 4.5e-4 us a row and column, half the rate of a large f32 product.)
        const int on = room / 256, widest = D == 256 ? 128 : 256;
        const float read = room * 64 * rb / 5.3e6f;
        const float products = dtype == ULLM_DT_F32
                                   ? on * s.rows() * D * 4.5e-4f
                                   : on * s.rows() * 1.35f * kTreeCost[0][D / 128][D == 256 ? 3 : 4].few / widest;
        float full = c.full;
        if (full > .9f * read && full < 1.25f * read)
            full = std::min(full, std::max({c.few, products, full / std::sqrt((float)row_tiles)}));
        const int64_t most = batch <= 256 ? std::min(room / units, batch * ((blocks + part) / part)) : 0;
        for (int64_t slots = batch, k = 1;;) {
            const float wgs = (float)slots * units / room;
            const float block = c.few + (full - c.few) * std::min(std::max((wgs - .125f) / .875f, 0.f), 1.f);
            // start and end of a workgroup: what is left at no keys of the times that kTreeCost
            // is the slope of (16 bits x 128, 16 to 256 rows: 4.4, 5.6, 7.3, 7.3, 10.9)
            float us = 4.5f + s.rows() * rb * 1e-4f;
            if (slots == batch) {
                us = std::max(wgs, 1.f) * (us + blocks * block);
            } else {
                // (the sequences of a batch are taken to have 0.75 max_len on average)
                const float len = std::ceil((batch > 1 ? .75f : 1.f) * blocks * batch / slots);
                us += std::max(len, (float)part) * block;
                // the merge, the cut, and the joined partials: 8 bytes an element at 6.6 TB/s
                us += 3 + (batch > 1 ? 1.5f : 0) + 1.2e-6f * slots * n_kv * rows * D;
            }
            if (us < least) {
                least = us;
                best.shape = s;
                best.plan = TreePlan{};
                best.plan.batch = batch, best.plan.n_kv = n_kv, best.plan.row_tiles = row_tiles;
                best.plan.least = part, best.plan.slots = (int)slots;
                best.rows = slots > batch ? slots * units * s.rows() : 0;
            }
            if (slots >= most) break;
            k += k < 4 ? 1 : (k & (k - 1)) ? k / 3 : k / 2;  // 1, 2, 3, 4, 6, 8, 12, ..
            slots = std::min(batch * k, most);
        }
        if (s.rows() == 16) return best;
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
