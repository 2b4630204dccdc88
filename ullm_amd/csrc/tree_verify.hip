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
    int vocab, max_nodes, distinct, batch;
    const int32_t *tokens, *parents, *n_nodes;
    const float *u;
    int32_t *path, *count, *next;
    int chunk, chunks, slices;  // entries of a chunk of a row, chunks of a row, workgroups of a sequence
    struct VerifyEnd *end;      // [batch]
    double *sums;               // [batch][chunks]: of what is left of the last row
};
// Where a sequence ends: the last node kept (-1: none), and c.
struct VerifyEnd {
    int cur, pad;
    double c;
};

constexpr int kVerifyMax = 1024;   // nodes of a tree
constexpr int kVerifyT = 1024, kVerifyW = kVerifyT / 64;
constexpr int kVerifySums = 1024;  // chunks of a row
constexpr int kVerifyChunk = 1024; // entries of a chunk, or a multiple: 16 a lane

// A probability: what is none (below 0, infinite, NaN) counts as 0.
__device__ __forceinline__ float prob(float x) { return __float_as_uint(x) < 0x7f800000u ? x : 0.f; }
// A random number of [0, 1).
__device__ __forceinline__ double unit(float u) { return fminf(fmaxf(u, 0.f), 0x1.fffffep-1f); }
// The part of p that the rejected drafts leave.
__device__ __forceinline__ double rest(float p, float q, double c) { return fmax(p - c * q, 0.); }

// Entry i of a row.
template <class T>
__device__ __forceinline__ float entry(const char *row, int i) {
    if constexpr (__is_same(T, F32)) return prob(((const float *)row)[i]);
    else if constexpr (__is_same(T, F16)) return prob((float)((const _Float16 *)row)[i]);
    else return prob(__uint_as_float((uint32_t)((const uint16_t *)row)[i] << 16));
}
// Entries of a row from i on, N of them, those past V as 0.  Rows begin at any element.
template <class T, int N>
__device__ __forceinline__ void entries(const char *row, int i, int V, float *o) {
    typedef u32x4 loose __attribute__((aligned(2)));
    constexpr int n = Chunk<T>::n;
    if (i + N <= V) {
        u32x4 x[N / n];
#pragma unroll
        for (int j = 0; j < N / n; j++) x[j] = *(const loose *)(row + (int64_t)(i + j * n) * T::bytes);
#pragma unroll
        for (int j = 0; j < N / n; j++) Chunk<T>::widen(x[j], o + j * n);
        // Most rows hold probabilities only, so what is none is looked for with one maximum
        // a value: 8 trees of 26 take 31.5 us so, 33.7 with every value put right (29 with none).
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < N; j++) top = max(top, __float_as_uint(o[j]));
        if (__any(top >= 0x7f800000u))
#pragma unroll
            for (int j = 0; j < N; j++) o[j] = prob(o[j]);
        return;
    }
#pragma unroll
    for (int j = 0; j < N; j++) o[j] = i + j < V ? entry<T>(row, i + j) : 0.f;
}

template <int CTRL, int ROWS, int BANKS>
__device__ __forceinline__ double dpp64(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)u, CTRL, ROWS, BANKS, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, ROWS, BANKS, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Inclusive sums over the lanes (row shifts, then the row broadcasts).
__device__ __forceinline__ double wave_scan64(double x) {
    x += dpp64<0x111, 0xf, 0xf>(x);
    x += dpp64<0x112, 0xf, 0xf>(x);
    x += dpp64<0x114, 0xf, 0xe>(x);
    x += dpp64<0x118, 0xf, 0xc>(x);
    x += dpp64<0x142, 0xa, 0xf>(x);
    x += dpp64<0x143, 0xc, 0xf>(x);
    return x;
}
__device__ __forceinline__ double lane64(double x, int l) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_readlane((int)u, l), hi = __builtin_amdgcn_readlane((int)(u >> 32), l);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// What is left of a row: R = max(p - c q, 0), or p without the tokens in `gone`.
template <class T>
struct Left {
    const char *p, *q;  // rows; q null: gone
    double c;
    const int *gone;    // in LDS
    int n_gone, V;
    // Entries i .. i + N - 1; the wave's are those of one chunk, from k0 on.
    template <int N>
    __device__ __forceinline__ void get(int i, int k0, int k1, double (&w)[N]) const {
        float x[N];
        entries<T, N>(p, i, V, x);
        if (q && c != 0.) {
            float y[N];
            entries<T, N>(q, i, V, y);
#pragma unroll
            for (int j = 0; j < N; j++) w[j] = rest(x[j], y[j], c);
            return;
        }
#pragma unroll
        for (int j = 0; j < N; j++) w[j] = x[j];
        for (int g = 0; g < n_gone; g++) {
            const int t = gone[g];
            if (t < k0 || t >= k1) continue;
#pragma unroll
            for (int j = 0; j < N; j++)
                if (t == i + j) w[j] = 0.;
        }
    }
    // Sum of a chunk of entries, in every lane.
    __device__ __forceinline__ double sum(int k, int chunk) const {
        const int lane = threadIdx.x & 63;
        double s = 0.;
        for (int k0 = k * chunk; k0 < min((k + 1) * chunk, V); k0 += kVerifyChunk) {
            constexpr int n = Chunk<T>::n;
            double w[16 / n][n];
#pragma unroll
            for (int j = 0; j < 16 / n; j++) get<n>(k0 + (j * 64 + lane) * n, k0, k0 + kVerifyChunk, w[j]);
#pragma unroll
            for (int j = 0; j < 16 / n; j++)
#pragma unroll
                for (int i = 0; i < n; i += 4) s += (w[j][i] + w[j][i + 1]) + (w[j][i + 2] + w[j][i + 3]);
        }
        return lane64(wave_scan64(s), 63);
    }
};

// The nodes of sequence b in order, and the chunk sums of what its last row leaves.
// `slices` workgroups a sequence: all of them walk (a few LDS reads a node, where no sum
// is asked for; a rejected node with siblings left asks for one, which each finds for
// itself: the rows are in L2 then), each sums its chunks, the first writes the path.  Bound by
// latency (the nodes, their probabilities, the walk, the row: 6.5 us) and by the 64-bit
// sums, 6 to 8 us for one of 100003 entries in a workgroup.  In one workgroup a
// sequence, with the token found in the same launch, 32 chains of 7 over 131072 tokens took
// 108 us in place of 17.5, 8 trees of 26 over 100003 115 in place of 31 to 55.
template <class T>
__global__ __launch_bounds__(kVerifyT) void verify_walk_kernel(VerifyArgs a) {
    __shared__ int parent[kVerifyMax], token[kVerifyMax], gone[kVerifyMax];
    __shared__ float pu[kVerifyMax], px[kVerifyMax], qx[kVerifyMax];
    __shared__ double part[2][kVerifyW];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int b = blockIdx.x % a.batch, slice = blockIdx.x / a.batch, V = a.vocab;
    const char *p = a.p + b * a.p_seq * T::bytes, *q = a.q ? a.q + b * a.q_seq * T::bytes : nullptr;
    const int n = a.n_nodes ? min(max(a.n_nodes[b], 0), a.max_nodes) : a.max_nodes;
    if (tid < n) {
        const int64_t at = (int64_t)b * a.max_nodes + tid;
        const int par = a.parents ? max(a.parents[at], -1) : tid - 1, x = a.tokens[at];
        const bool ok = par < tid && x >= 0 && x < V;
        parent[tid] = ok ? par : kVerifyMax;  // no node goes on from there
        token[tid] = x;
        pu[tid] = (float)unit(a.u[(int64_t)b * (a.max_nodes + 1) + tid]);
        px[tid] = ok ? entry<T>(p + (int64_t)(par + 1) * a.p_row * T::bytes, x) : 0.f;
        qx[tid] = ok && q ? entry<T>(q + (int64_t)(par + 1) * a.q_row * T::bytes, x) : 0.f;
    }
    __syncthreads();
    int cur = -1, kept = 0, flip = 0;
    double mass = 1., left = 1.;
    Left<T> l{p, q, 0., gone, 0, V};
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
                for (int g = 0; g < l.n_gone; g++)
                    if (gone[g] == token[i1]) r = 0.;
                keep = r > 0. && pu[i1] * mass < r;
                if (!keep) {
                    mass = fmax(mass - r, 0.);
                    if (tid == 0) gone[l.n_gone] = token[i1];
                    l.n_gone++;
                    __syncthreads();
                }
            } else {
                if (stale) {  // the sum over the whole row
                    double s = 0.;
                    for (int k = wave; k < a.chunks; k += kVerifyW) s += l.sum(k, a.chunk);
                    if (lane == 0) part[flip][wave] = s;
                    __syncthreads();
                    mass = 0.;
                    for (int w = 0; w < kVerifyW; w++) mass += part[flip][w];
                    flip ^= 1;
                    stale = false;
                }
                if (l.c != 0.) r = rest(px[i1], qx[i1], l.c);
                keep = r > 0. && pu[i1] * (qx[i1] / left) * mass < r;
                if (!keep) {
                    l.c += mass / left;
                    if (a.distinct) left = fmax(left - qx[i1], 0x1p-24);
                    stale = true;
                }
            }
            if (keep) {
                cur = i1;
                if (slice == 0 && tid == 0) a.path[(int64_t)b * a.max_nodes + kept] = i1;
                kept++;
                l.n_gone = 0, l.c = 0., mass = 1., left = 1., stale = false;
                l.p = p + (int64_t)(i1 + 1) * a.p_row * T::bytes;
                l.q = q ? q + (int64_t)min(i1 + 1, a.max_nodes - 1) * a.q_row * T::bytes : nullptr;
                __syncthreads();
            }
        }
    }
    for (int k = slice * kVerifyW + wave; k < a.chunks; k += a.slices * kVerifyW) {
        const double s = l.sum(k, a.chunk);
        if (lane == 0) a.sums[(int64_t)b * a.chunks + k] = s;
    }
    if (slice) return;
    for (int i = kept + tid; i < a.max_nodes; i += kVerifyT) a.path[(int64_t)b * a.max_nodes + i] = -1;
    if (tid == 0) {
        a.count[b] = kept;
        a.end[b] = VerifyEnd{cur, 0, l.c};
    }
}

// The token that follows: the first whose cumulative sum exceeds u times the whole; its
// chunk by the chunks' sums, then itself.  A workgroup a sequence.
template <class T>
__global__ __launch_bounds__(kVerifyT) void verify_next_kernel(VerifyArgs a) {
    __shared__ int gone[kVerifyMax], n_gone, where;
    __shared__ double part[kVerifyW], base;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), b = blockIdx.x, V = a.vocab;
    const VerifyEnd e = a.end[b];
    double mine = tid < a.chunks ? a.sums[(int64_t)b * a.chunks + tid] : 0.;
    const double u = unit(a.u[(int64_t)b * (a.max_nodes + 1) + a.max_nodes]);
    Left<T> l{a.p + (b * a.p_seq + (e.cur + 1) * a.p_row) * T::bytes,
              a.q ? a.q + (b * a.q_seq + min(e.cur + 1, a.max_nodes - 1) * a.q_row) * T::bytes : nullptr, e.c, gone, 0, V};
    if (tid == 0) n_gone = 0, where = -1;
    __syncthreads();
    if (!a.q) {  // every child of the last node kept has been rejected
        const int n = a.n_nodes ? min(max(a.n_nodes[b], 0), a.max_nodes) : a.max_nodes;
        if (tid > e.cur && tid < n) {
            const int64_t at = (int64_t)b * a.max_nodes + tid;
            const int x = a.tokens[at];
            if ((a.parents ? max(a.parents[at], -1) : tid - 1) == e.cur && x >= 0 && x < V) gone[atomicAdd(&n_gone, 1)] = x;
        }
        __syncthreads();
        l.n_gone = n_gone;
    }
    // sums of the chunks before each thread's, and the whole
    double before, total;
    auto scan = [&]() __attribute__((always_inline)) {
        const double s = wave_scan64(mine);
        __syncthreads();
        if (lane == 63) part[wave] = s;
        __syncthreads();
        before = s - mine, total = 0.;
        for (int w = 0; w < kVerifyW; w++) {
            if (w < wave) before += part[w];
            total += part[w];
        }
    };
    scan();
    if (!(total > 0.)) {  // nothing is left: the target's own
        l.c = 0., l.n_gone = 0;
        __shared__ double again[kVerifySums];
        for (int k = wave; k < a.chunks; k += kVerifyW) {
            const double s = l.sum(k, a.chunk);
            if (lane == 0) again[k] = s;
        }
        __syncthreads();
        mine = tid < a.chunks ? again[tid] : 0.;
        scan();
    }
    if (!(total > 0.)) {
        if (tid == 0) a.next[b] = -1;
        return;
    }
    const double at = u * total;
    if (mine > 0. && before + mine > at) atomicMax(&where, kVerifySums - tid);  // the lowest
    __syncthreads();
    const int k = kVerifySums - where;
    if (tid == k) base = before;
    __syncthreads();
    if (wave) return;
    double sum = base;
    int last = -1;
    for (int k0 = k * a.chunk; k0 < min((k + 1) * a.chunk, V); k0 += kVerifyChunk) {
        double w[16], s = 0.;
        l.template get<16>(k0 + lane * 16, k0, k0 + kVerifyChunk, w);
#pragma unroll
        for (int j = 0; j < 16; j++) s += w[j];
        const double upto = wave_scan64(s);
        double x = sum + (upto - s);  // before this lane's entries
        int hit = -1, some = -1;
#pragma unroll
        for (int j = 0; j < 16; j++) {
            x += w[j];
            if (w[j] > 0.) {
                some = j;
                if (hit < 0 && x > at) hit = j;
            }
        }
        const uint64_t hits = __ballot(hit >= 0), any = __ballot(some >= 0);
        if (any) {
            const int from = 63 - __builtin_clzll(any);
            last = k0 + from * 16 + __builtin_amdgcn_readlane(some, from);
        }
        if (hits) {
            const int from = __builtin_ctzll(hits);
            last = k0 + from * 16 + __builtin_amdgcn_readlane(hit, from);
            break;
        }
        sum += lane64(upto, 63);
    }
    if (lane == 0) a.next[b] = last;
}

}  // namespace ullm

using namespace ullm;

static bool overlap(const void *a, size_t na, const void *b, size_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a && b && na && nb && x < y + nb && y < x + na;
}

static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

extern "C" size_t ullm_hip_tree_verify_workspace_bytes(int vocab, int batch) {
    if (vocab < 1 || vocab > 1 << 30 || batch < 1) return 0;
    const int64_t chunks = std::min<int64_t>(kVerifySums, ((int64_t)vocab + kVerifyChunk - 1) / kVerifyChunk);
    return up256((size_t)batch * sizeof(VerifyEnd)) + (size_t)batch * chunks * sizeof(double);
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
    const int chunk = kVerifyChunk * ((vocab + kVerifyChunk * kVerifySums - 1) / (kVerifyChunk * kVerifySums));
    const int chunks = (vocab + chunk - 1) / chunk;
    // workgroups of a sequence: a chunk a wave, two workgroups a CU
    const int slices = std::max(1, std::min((chunks + kVerifyW - 1) / kVerifyW, 512 / batch));
    const VerifyArgs a{(const char *)target, max_nodes ? (const char *)draft : nullptr, target_seq, target_row, draft_seq,
                       draft_row, vocab, max_nodes, distinct != 0, batch, tokens, parents, n_nodes, uniform, path, n_accept, next,
                       chunk, chunks, slices, (VerifyEnd *)workspace,
                       (double *)((char *)workspace + up256((size_t)batch * sizeof(VerifyEnd)))};
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid(batch * slices), block(kVerifyT);
    auto launch = [&](auto walk, auto last) {
        launch_kernel(walk, grid, block, 0, st, a);
        launch_kernel(last, dim3(batch), block, 0, st, a);
    };
    if (dtype == ULLM_DT_F32) launch(verify_walk_kernel<F32>, verify_next_kernel<F32>);
    else if (dtype == ULLM_DT_F16) launch(verify_walk_kernel<F16>, verify_next_kernel<F16>);
    else launch(verify_walk_kernel<BF16>, verify_next_kernel<BF16>);
    return check_hip(hipGetLastError(), "tree_verify launch");
}
