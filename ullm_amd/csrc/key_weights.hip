// The attention weight that the keys of a cache get from some rows of queries:
// ullm_hip_key_weights(_paged).
#include <algorithm>
#include <climits>
#include "common.hpp"
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
    float2 *ml;  // [batch][n_kv][max_rows * gq]: largest score and sum of exp2 of each row
};

template <class T>
__device__ __forceinline__ void load16(const void *p, float *o) {
    Chunk<T>::widen(ld16(p), o);
}

// Byte offset of key t of sequence b; -1: its page is none of the pool's.
__device__ __forceinline__ int64_t key_row(const WeightArgs &a, int b, int t) {
    if (!a.tab) return b * a.seq_b + t * a.rb;
    const int phys = a.tab[(int64_t)b * a.tab_stride + (t >> a.shift)];
    if (phys < 0 || phys >= a.n_pages) return -1;
    return (((int64_t)phys << a.shift) + (t & ((1 << a.shift) - 1))) * a.rb;
}

template <class TK, int D>
__device__ __forceinline__ float key_dot(const WeightArgs &a, const float *q, int b, int g, int t) {
    const int64_t at = key_row(a, b, t);
    if (at < 0) return 0.f;
    const char *p = a.k + at + (int64_t)g * D * TK::bytes;
    float s = 0.f;
#pragma unroll 4
    for (int c = 0; c < D; c += Chunk<TK>::n) {
        float x[Chunk<TK>::n];
        load16<TK>(p + c * TK::bytes, x);
#pragma unroll
        for (int i = 0; i < Chunk<TK>::n; i++) s = fmaf(x[i], q[c + i], s);
    }
    return s;
}

// Largest score and sum of one row, a workgroup a row.
template <class TQ, class TK, int D>
__global__ __launch_bounds__(256) void weight_rows_kernel(WeightArgs a) {
    __shared__ float q[D], sm[4], sl[4];
    const int tid = threadIdx.x, b = blockIdx.z, h = blockIdx.y, i = blockIdx.x, g = h / a.gq;
    const int len = min(max(a.len[b], 0), a.max_len), n = a.n_rows ? min(max(a.n_rows[b], 0), a.max_rows) : a.max_rows;
    const int pos = len - n + i;
    if (i >= n || pos < 0) return;
    if (tid < D / Chunk<TQ>::n) {
        const char *p = (const char *)a.q + (((int64_t)b * a.max_rows + i) * a.n_head + h) * D * TQ::bytes;
        load16<TQ>(p + tid * 16, q + tid * Chunk<TQ>::n);
    }
    __syncthreads();
    const int t0 = a.window ? max(0, pos + 1 - a.window) : 0;
    float m = -INFINITY, l = 0.f;
    for (int t = t0 + tid; t <= pos; t += 256) {
        const float s = key_dot<TK, D>(a, q, b, g, t) * a.qs;
        if (s > m) l *= exp2f(m - s), m = s;
        l += s == m ? 1.f : exp2f(s - m);
    }
    const float wm = wave_max(m);
    l = wave_sum(m == -INFINITY ? l : l * exp2f(m - wm));
    if ((tid & 63) == 0) sm[tid >> 6] = wm, sl[tid >> 6] = l;
    __syncthreads();
    if (tid) return;
    const float bm = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    float bl = 0.f;
    for (int w = 0; w < 4; w++) bl += sm[w] == -INFINITY ? sl[w] : sl[w] * exp2f(sm[w] - bm);
    a.ml[((int64_t)b * a.n_kv + g) * a.max_rows * a.gq + (int64_t)i * a.gq + h % a.gq] = float2{bm, bl};
}

// Weights of the keys of one kv head, a thread a key.
template <class TQ, class TK, int D>
__global__ __launch_bounds__(256) void weight_keys_kernel(WeightArgs a) {
    __shared__ float q[D];
    const int tid = threadIdx.x, b = blockIdx.z, g = blockIdx.y, t = blockIdx.x * 256 + tid;
    const int len = min(max(a.len[b], 0), a.max_len), n = a.n_rows ? min(max(a.n_rows[b], 0), a.max_rows) : a.max_rows;
    if ((int)blockIdx.x * 256 >= len) return;
    float sum = 0.f;
    for (int i = max(0, (int)blockIdx.x * 256 - (len - n)); i < n; i++) {
        const int pos = len - n + i;
        if (pos < 0) continue;
        for (int h = 0; h < a.gq; h++) {
            __syncthreads();
            if (tid < D / Chunk<TQ>::n) {
                const char *p = (const char *)a.q + (((int64_t)b * a.max_rows + i) * a.n_head + g * a.gq + h) * D * TQ::bytes;
                load16<TQ>(p + tid * 16, q + tid * Chunk<TQ>::n);
            }
            __syncthreads();
            if (t <= pos && (!a.window || t > pos - a.window)) {
                const float2 ml = a.ml[((int64_t)b * a.n_kv + g) * a.max_rows * a.gq + (int64_t)i * a.gq + h];
                const float s = key_dot<TK, D>(a, q, b, g, t) * a.qs;
                sum += exp2f(s - ml.x) / ml.y;
            }
        }
    }
    if (t >= len) return;
    float *w = a.w + ((int64_t)b * a.n_kv + g) * a.w_stride + t;
    *w = a.decay == 0.f ? sum : fmaf(a.decay, *w, sum);
}

static size_t weights_ws(int batch, int max_rows, int n_head) { return (size_t)batch * max_rows * n_head * sizeof(float2); }

template <class TQ, class TK, int D>
static void launch_weights(const WeightArgs &a, hipStream_t st) {
    if (a.max_rows) launch_kernel(weight_rows_kernel<TQ, TK, D>, dim3(a.max_rows, a.n_head, a.batch), dim3(256), 0, st, a);
    launch_kernel(weight_keys_kernel<TQ, TK, D>, dim3((a.max_len + 255) / 256, a.n_kv, a.batch), dim3(256), 0, st, a);
}
template <class TQ, class TK>
static void launch_weights(const WeightArgs &a, int D, hipStream_t st) {
    if (D == 64) launch_weights<TQ, TK, 64>(a, st);
    else if (D == 128) launch_weights<TQ, TK, 128>(a, st);
    else launch_weights<TQ, TK, 256>(a, st);
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
    if ((int64_t)a.max_rows * a.n_head > 1 << 23) return set_error(ULLM_HIP_E_INVALID, "%s: too many rows", fn);
    if (kv_stride < (int64_t)a.n_kv * head_dim || a.w_stride < a.max_len)
        return set_error(ULLM_HIP_E_INVALID, "%s: kv_stride or weights_stride too small", fn);
    if (a.batch == 0 || a.max_len == 0) return ULLM_HIP_OK;
    if ((!a.q && a.max_rows) || !a.k || !a.len || !a.w) return set_error(ULLM_HIP_E_INVALID, "%s: null tensor pointer", fn);
    const int eb = dtype_bytes(dtype);
    if (((uintptr_t)a.q | (uintptr_t)a.k) & 15 || kv_stride * eb % 16 || a.seq_b % 16)
        return set_error(ULLM_HIP_E_INVALID, "%s: tensors and row strides must be 16-byte aligned", fn);
    const size_t need = weights_ws(a.batch, a.max_rows, a.n_head);
    if (need && (!ws || ws_bytes < need || (uintptr_t)ws & 255))
        return set_error(ULLM_HIP_E_WORKSPACE, "%s: workspace of %zu bytes, 256-byte aligned, needed", fn, need);
    a.gq = a.n_head / a.n_kv;
    a.qs = scale * kLog2e;
    a.rb = kv_stride * eb;
    a.ml = (float2 *)ws;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == ULLM_DT_F32) launch_weights<F32, F32>(a, head_dim, st);
    else if (dtype == ULLM_DT_F16) q_dtype == dtype ? launch_weights<F16, F16>(a, head_dim, st) : launch_weights<F32, F16>(a, head_dim, st);
    else q_dtype == dtype ? launch_weights<BF16, BF16>(a, head_dim, st) : launch_weights<F32, BF16>(a, head_dim, st);
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
                       decay, weights, weights_stride, nullptr};
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
                       weights_stride, nullptr};
    return key_weights("key_weights_paged", a, q_dtype, kv_dtype, kv_stride, head_dim, scale, workspace,
                       workspace_bytes, stream);
}

extern "C" size_t ullm_hip_key_weights_workspace_bytes(int kv_dtype, int batch, int max_rows, int max_len, int window,
                                                       int n_head, int n_kv_head, int head_dim) {
    if (!dtype_ok(kv_dtype) || (head_dim != 64 && head_dim != 128 && head_dim != 256) || batch < 1 || max_rows < 1 ||
        max_len < 1 || window < 0 || n_head < 1 || n_kv_head < 1 || n_head % n_kv_head || n_head > 65535 ||
        (int64_t)max_rows * n_head > 1 << 23)
        return 0;
    return weights_ws(batch, max_rows, n_head);
}
