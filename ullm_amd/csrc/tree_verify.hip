// Which nodes of drafted trees are kept, from the target's probabilities, the
// draft's and given random numbers, and the token that follows:
// ullm_hip_tree_verify.
#include <algorithm>
#include <climits>
#include "common.hpp"
#include "wave.hpp"

namespace ullm {

struct VerifyArgs {
    const char *p, *q;  // q null: drafts without probabilities
    int64_t p_seq, p_row, q_seq, q_row;  // elements from sequence to sequence, from row to row
    int vocab, max_nodes, distinct;
    const int32_t *tokens, *parents, *n_nodes;
    const float *u;
    int32_t *path, *count, *next;
};

constexpr int kVerifyMax = 1024;   // nodes of a tree
constexpr int kVerifyT = 1024;
constexpr int kVerifySums = 1024;  // chunks of a row

// A probability: what is none (below 0, NaN, infinite) counts as 0.
template <class T>
__device__ __forceinline__ float prob(const char *row, int i) {
    float x;
    if constexpr (__is_same(T, F32)) x = ((const float *)row)[i];
    else if constexpr (__is_same(T, F16)) x = (float)((const _Float16 *)row)[i];
    else x = __uint_as_float((uint32_t)((const uint16_t *)row)[i] << 16);
    return x > 0.f && x <= 3.4028234e38f ? x : 0.f;
}
// A random number of [0, 1).
__device__ __forceinline__ double unit(float u) { return fminf(fmaxf(u, 0.f), 0x1.fffffep-1f); }

// The part of p that the rejected drafts leave: max(p - c q, 0).
__device__ __forceinline__ double rest(float p, float q, double c) { return fmax(p - c * q, 0.); }

__device__ __forceinline__ double wave_sum64(double x) {
#pragma unroll
    for (int o = 1; o < 64; o *= 2) x += __shfl_xor(x, o);
    return x;
}
__device__ __forceinline__ double wave_scan64(double x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const double y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    return x;
}

// One workgroup a sequence.
template <class T>
__global__ __launch_bounds__(kVerifyT) void verify_kernel(VerifyArgs a) {
    __shared__ int parent[kVerifyMax], token[kVerifyMax], gone[kVerifyMax];
    __shared__ float pu[kVerifyMax], px[kVerifyMax], qx[kVerifyMax];
    __shared__ double sums[kVerifySums], part[kVerifyT / 64];
    __shared__ int where;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x, V = a.vocab;
    const char *p = a.p + b * a.p_seq * T::bytes, *q = a.q ? a.q + b * a.q_seq * T::bytes : nullptr;
    const int n = a.n_nodes ? min(max(a.n_nodes[b], 0), a.max_nodes) : a.max_nodes;
    for (int i = tid; i < n; i += kVerifyT) {
        const int64_t at = (int64_t)b * a.max_nodes + i;
        const int par = a.parents ? max(a.parents[at], -1) : i - 1, x = a.tokens[at];
        const bool ok = par < i && x >= 0 && x < V;
        parent[i] = ok ? par : kVerifyMax;  // no node goes on from there
        token[i] = x;
        pu[i] = (float)unit(a.u[(int64_t)b * (a.max_nodes + 1) + i]);
        px[i] = ok ? prob<T>(p + (int64_t)(par + 1) * a.p_row * T::bytes, x) : 0.f;
        qx[i] = ok && q ? prob<T>(q + (int64_t)(par + 1) * a.q_row * T::bytes, x) : 0.f;
    }
    __syncthreads();
    const int chunk = 512 * ((V + 512 * kVerifySums - 1) / (512 * kVerifySums)), chunks = (V + chunk - 1) / chunk;
    int n_gone = 0, cur = -1, kept = 0;
    double c = 0., mass = 1., left = 1.;
    const char *pr = p, *qr = q;
    // an element of what is left of the current row
    auto weight = [&](int i) -> double {
        const float x = prob<T>(pr, i);
        if (q) return c == 0. ? (double)x : rest(x, prob<T>(qr, i), c);
        for (int j = 0; j < n_gone; j++)
            if (gone[j] == i) return 0.;
        return x;
    };
    // its sums over chunks, and the whole
    auto all = [&]() -> double {
        __syncthreads();
        for (int k = wave; k < chunks; k += kVerifyT / 64) {
            double s = 0.;
            for (int i = k * chunk + lane; i < min((k + 1) * chunk, V); i += 64) s += weight(i);
            s = wave_sum64(s);
            if (lane == 0) sums[k] = s;
        }
        __syncthreads();
        double s = wave_sum64(tid < chunks ? sums[tid] : 0.);
        if (lane == 0) part[wave] = s;
        __syncthreads();
        s = 0.;
        for (int w = 0; w < kVerifyT / 64; w++) s += part[w];
        return s;
    };
    bool stale = false;  // mass is that of an earlier c
    for (int i0 = 0; i0 < n; i0 += 64) {
        for (int done = 0; done < 64;) {
            const int i = i0 + lane;
            const uint64_t m = __ballot(i < n && parent[i] == cur) >> done << done;
            if (!m) break;
            const int j = __builtin_ctzll(m), i1 = i0 + j;
            done = j + 1;
            bool keep;
            double r = px[i1];
            if (!q) {
                for (int g = 0; g < n_gone; g++)
                    if (gone[g] == token[i1]) r = 0.;
                keep = r > 0. && pu[i1] * mass < r;
                if (!keep) {
                    mass = fmax(mass - r, 0.);
                    if (tid == 0) gone[n_gone] = token[i1];
                    n_gone++;
                    __syncthreads();
                }
            } else {
                if (stale) mass = all(), stale = false;
                if (c != 0.) r = rest(px[i1], qx[i1], c);
                keep = r > 0. && pu[i1] * (qx[i1] / left) * mass < r;
                if (!keep) {
                    c += mass / left;
                    if (a.distinct) left = fmax(left - qx[i1], 0x1p-24);
                    stale = true;
                }
            }
            if (keep) {
                cur = i1;
                if (tid == 0) a.path[(int64_t)b * a.max_nodes + kept] = i1;
                kept++;
                n_gone = 0, c = 0., mass = 1., left = 1., stale = false;
                pr = p + (int64_t)(i1 + 1) * a.p_row * T::bytes;
                qr = q ? q + (int64_t)min(i1 + 1, a.max_nodes - 1) * a.q_row * T::bytes : nullptr;
                __syncthreads();
            }
        }
    }
    for (int i = kept + tid; i < a.max_nodes; i += kVerifyT) a.path[(int64_t)b * a.max_nodes + i] = -1;
    double total = all();
    if (!(total > 0.)) {  // nothing is left: the target's own
        n_gone = 0, c = 0.;
        total = all();
    }
    if (tid == 0) a.count[b] = kept;
    if (!(total > 0.)) {
        if (tid == 0) a.next[b] = -1;
        return;
    }
    const double u = unit(a.u[(int64_t)b * (a.max_nodes + 1) + a.max_nodes]);
    // the first token whose cumulative sum exceeds u times the whole: its chunk, then itself
    const double mine = tid < chunks ? sums[tid] : 0., s = wave_scan64(mine);
    __syncthreads();
    if (lane == 63) part[wave] = s;
    if (tid == 0) where = -1;
    __syncthreads();
    double before = s - mine;
    for (int w = 0; w < wave; w++) before += part[w];
    total = 0.;
    for (int w = 0; w < kVerifyT / 64; w++) total += part[w];
    const double at = u * total;
    if (mine > 0. && before + mine > at) atomicMax(&where, kVerifySums - tid);  // the lowest
    __syncthreads();
    const int k = kVerifySums - where;
    if (tid == k) part[0] = before;
    __syncthreads();
    if (wave) return;
    double base = part[0];
    int last = -1;
    for (int i0 = k * chunk; i0 < min((k + 1) * chunk, V); i0 += 64) {
        const double w = i0 + lane < V ? weight(i0 + lane) : 0., t = wave_scan64(w);
        const uint64_t hit = __ballot(w > 0. && base + t > at), some = __ballot(w > 0.);
        if (some) last = i0 + 63 - __builtin_clzll(some);
        if (hit) {
            last = i0 + __builtin_ctzll(hit);
            break;
        }
        base += __shfl(t, 63);
    }
    if (lane == 0) a.next[b] = last;
}

}  // namespace ullm

using namespace ullm;

static bool overlap(const void *a, size_t na, const void *b, size_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a && b && na && nb && x < y + nb && y < x + na;
}

extern "C" size_t ullm_hip_tree_verify_workspace_bytes(int vocab, int batch) {
    return vocab < 1 || batch < 1 ? 0 : 256;
}

extern "C" int ullm_hip_tree_verify(const void *target, int64_t target_seq, int64_t target_row, const void *draft,
                                    int64_t draft_seq, int64_t draft_row, int dtype, int vocab, const int32_t *tokens,
                                    const int32_t *parents, const int32_t *n_nodes, const float *uniform, int max_nodes,
                                    int distinct, int batch, int32_t *path, int32_t *n_accept, int32_t *next,
                                    void *workspace, size_t workspace_bytes, void *stream) {
    if (!dtype_ok(dtype)) return set_error(ULLM_HIP_E_UNSUPPORTED, "tree_verify: dtype %d", dtype);
    if (batch < 0 || batch > 65535 || max_nodes < 0 || max_nodes > kVerifyMax || vocab < 1 || vocab > 1 << 30)
        return set_error(ULLM_HIP_E_INVALID, "tree_verify: batch %d not in 0..65535, max_nodes %d not in 0..%d or vocab %d not in 1..2^30",
                         batch, max_nodes, kVerifyMax, vocab);
    if (target_seq < 0 || target_row < 0 || draft_seq < 0 || draft_row < 0)
        return set_error(ULLM_HIP_E_INVALID, "tree_verify: strides below 0");
    if (batch == 0) return ULLM_HIP_OK;
    if (!target || !uniform || !n_accept || !next || (max_nodes && (!tokens || !path)))
        return set_error(ULLM_HIP_E_INVALID, "tree_verify: null tensor pointer");
    const uintptr_t mask = dtype_bytes(dtype) - 1;
    if (((uintptr_t)target | (uintptr_t)draft) & mask)
        return set_error(ULLM_HIP_E_INVALID, "tree_verify: target and draft must be aligned to their elements");
    const size_t nb = 4 * (size_t)batch, nn = nb * max_nodes;
    const void *outs[3] = {path, n_accept, next}, *ins[4] = {tokens, parents, n_nodes, uniform};
    const size_t no[3] = {nn, nb, nb}, ni[4] = {nn, nn, nb, nn + nb};
    for (int i = 0; i < 3; i++) {
        for (int j = 0; j < 4; j++)
            if (overlap(outs[i], no[i], ins[j], ni[j]))
                return set_error(ULLM_HIP_E_INVALID, "tree_verify: an output overlaps an input");
        for (int j = 0; j < i; j++)
            if (overlap(outs[i], no[i], outs[j], no[j]))
                return set_error(ULLM_HIP_E_INVALID, "tree_verify: the outputs overlap");
    }
    const size_t need = ullm_hip_tree_verify_workspace_bytes(vocab, batch);
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace & 255)
        return set_error(ULLM_HIP_E_WORKSPACE, "tree_verify: workspace of %zu bytes, 256-byte aligned, needed", need);
    const VerifyArgs a{(const char *)target, max_nodes ? (const char *)draft : nullptr, target_seq, target_row, draft_seq,
                       draft_row, vocab, max_nodes, distinct != 0, tokens, parents, n_nodes, uniform, path, n_accept, next};
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid(batch), block(kVerifyT);
    if (dtype == ULLM_DT_F32) launch_kernel(verify_kernel<F32>, grid, block, 0, st, a);
    else if (dtype == ULLM_DT_F16) launch_kernel(verify_kernel<F16>, grid, block, 0, st, a);
    else launch_kernel(verify_kernel<BF16>, grid, block, 0, st, a);
    return check_hip(hipGetLastError(), "tree_verify launch");
}
