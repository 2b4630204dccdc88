// Attention of a batch of drafted trees over the cache that holds their
// sequences (ullm_hip_attn_tree, ullm_hip_attn_tree_paged).
//
// Node i of sequence b, at position p_i, sees keys t < len_b (the sequence's
// own; with a window W those with t > p_i - W) and of the keys len_b + j the
// nodes j whose bit its mask has (p_j > p_i - W):
//   out[b,i,h] = sum_t softmax_t(scale * q[b,i,h] . K[t]) V[t]
// over those, and zeros where there is none or i >= n_b.
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
    float qs;  // scale * log2(e)
    void *out;
};

template <class T>
__device__ __forceinline__ float load1(const void *p, int64_t i) {
    if constexpr (__is_same(T, F32)) return ((const float *)p)[i];
    else if constexpr (__is_same(T, F16)) return (float)((const _Float16 *)p)[i];
    else return bf16_lo(((const uint16_t *)p)[i]);
}

// One wave per node and head, key by key.
template <class T, int D, int ODT>
__global__ __launch_bounds__(64) void tree_simple_kernel(TreeArgs a, TreeKv kv) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x, head = blockIdx.x, i = blockIdx.y, b = blockIdx.z;
    const int64_t row = ((int64_t)b * a.nodes + i) * a.n_head + head;
    const int n = a.n ? min(max(a.n[b], 0), a.nodes) : a.nodes;
    float o[E], q[E], m = -INFINITY, l = 0.f;
    for (int e = 0; e < E; e++) o[e] = 0.f, q[e] = load1<T>(a.q, row * D + lane * E + e) * a.qs;
    if (i < n) {
        const int len = min(max(a.len[b], 0), a.max_len), end = min(len + n, a.max_len);
        const int p = a.pos ? a.pos[(int64_t)b * a.nodes + i] : len + i;
        for (int t = 0; t < end; t++) {
            const int j = t - len;
            int kp = t;
            if (j >= 0) {
                const uint32_t w = a.mask ? a.mask[((int64_t)b * a.nodes + i) * a.words + (j >> 5)] : 0;
                if (a.mask ? !(w >> (j & 31) & 1) : j > i) continue;
                if (a.pos) kp = a.pos[(int64_t)b * a.nodes + j];
            }
            if (a.window > 0 && (int64_t)kp <= (int64_t)p - a.window) continue;
            int64_t at = b * kv.seq_b + t * kv.rb;
            bool ok = true;
            if (kv.tab) {
                const int pg = t >> kv.shift, phys = pg < kv.tab_stride ? kv.tab[(int64_t)b * kv.tab_stride + pg] : -1;
                ok = phys >= 0 && phys < kv.n_pages;
                at = (((int64_t)phys << kv.shift) + (t & ((1 << kv.shift) - 1))) * kv.rb;
            }
            const int64_t e0 = (int64_t)(head / a.kv_mul) * D + lane * E;
            float s = 0.f, v[E];
            for (int e = 0; e < E; e++) {
                s += ok ? q[e] * load1<T>(kv.k + at, e0 + e) : 0.f;
                v[e] = ok ? load1<T>(kv.v + at, e0 + e) : 0.f;
            }
            s = wave_sum(s);
            const float mn = fmaxf(m, s), mu = mn == -INFINITY ? 0.f : mn;
            const float c = __builtin_amdgcn_exp2f(m - mu), w = __builtin_amdgcn_exp2f(s - mu);
            l = l * c + w;
            for (int e = 0; e < E; e++) o[e] = o[e] * c + w * v[e];
            m = mn;
        }
    }
    for (int e = 0; e < E; e++) {
        const float x = l == 0.f ? 0.f : o[e] / l;  // a NaN score: NaN
        const int64_t at = row * D + lane * E + e;
        if (ODT == ULLM_DT_F32) ((float *)a.out)[at] = x;
        else ((uint16_t *)a.out)[at] = ODT == ULLM_DT_F16 ? f32_to_f16_bits(x) : f32_to_bf16_bits(x);
    }
}

template <class T, int D, int ODT>
static void launch_tree(const TreeArgs &a, const TreeKv &kv, int batch, hipStream_t st) {
    launch_kernel(tree_simple_kernel<T, D, ODT>, dim3(a.n_head, a.nodes, batch), dim3(64), 0, st, a, kv);
}
template <class T, int D>
static void launch_tree_out(int odt, int dt, const TreeArgs &a, const TreeKv &kv, int batch, hipStream_t st) {
    if (odt == ULLM_DT_F32) launch_tree<T, D, ULLM_DT_F32>(a, kv, batch, st);
    else if constexpr (__is_same(T, F16)) launch_tree<T, D, ULLM_DT_F16>(a, kv, batch, st);
    else if constexpr (__is_same(T, BF16)) launch_tree<T, D, ULLM_DT_BF16>(a, kv, batch, st);
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
    a.qs = scale * kLog2e;
    kv.rb = kv_stride * eb;
    hipStream_t st = (hipStream_t)stream;
    auto by_dim = [&](auto tc) {
        using T = decltype(tc);
        if (head_dim == 64) launch_tree_out<T, 64>(out_dtype, dtype, a, kv, batch, st);
        else if (head_dim == 128) launch_tree_out<T, 128>(out_dtype, dtype, a, kv, batch, st);
        else launch_tree_out<T, 256>(out_dtype, dtype, a, kv, batch, st);
    };
    if (dtype == ULLM_DT_F32) by_dim(F32{});
    else if (dtype == ULLM_DT_F16) by_dim(F16{});
    else by_dim(BF16{});
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
                     0.f, out};
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
                     0.f, out};
    const TreeKv kv{(const char *)k_pages, (const char *)v_pages, 0, 0, block_table, table_stride,
                    __builtin_ctz(page_size), n_pages};
    return attn_tree("attn_tree_paged", a, kv, dtype, kv_stride, batch, n_kv_head, head_dim, scale, out_dtype,
                     workspace, workspace_bytes, stream);
}

extern "C" size_t ullm_hip_tree_workspace_bytes(int dtype, int batch, int max_nodes, int max_len, int window,
                                                int n_head, int n_kv_head, int head_dim) {
    return 0;
}
