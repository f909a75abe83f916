// beam.cu -- beam search's selection: log-softmax of every beam's logits, added to the beam's score,
// and the k best (beam, token) pairs of each group of beams.
//
// The reference samples one token per sequence on the host (core/src/inference.cpp:2127-2244).
// Candidate (b, t) scores s_b + (x_bt - lse_b), lse_b = log sum_t exp x_bt.  Within a beam the order
// of the candidates is that of the logits (exact: no rounding decides it), so each beam contributes
// at most its k largest logits, which need no lse to be found: one pass over the logits does both.
// Across beams the scores are compared in 64 bits.
//
// beam_rows_kernel reads every logit once, in tiles of BEAM_TILE, cut into equal ranges of tiles per
// CTA whatever row they lie in.  Per part of a row that a CTA meets it leaves the part's k largest
// logits and its (max, sum of exp).  beam_merge_kernel, one CTA per group, joins the parts.
#include <math.h>

#include "../../include/dcgpu.h"
#include "common.cuh"
#include "kernels.h"

namespace dcg {

constexpr int BEAM_THREADS = 256;
constexpr int BEAM_WARPS = BEAM_THREADS / 32;
constexpr int BEAM_PER = 16;                             // logits per thread and tile
constexpr int BEAM_TILE = BEAM_THREADS * BEAM_PER;
constexpr int BEAM_CTAS = 5;                             // resident CTAs per SM (33 KB of keys each)
constexpr int BEAM_RANK = 256;                           // lists up to this long are sorted by counting
constexpr int BEAM_LIMIT = BEAM_RANK - 64;               // a list that grew this long is pruned
constexpr int BEAM_CAP = BEAM_LIMIT + BEAM_TILE;         // a whole tile always fits
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// order-preserving key of a logit and its token: larger logit first, then the lower token; 0 = none
__device__ __forceinline__ uint64_t beam_key(float x, uint32_t token) {
    const uint32_t u = __float_as_uint(x + 0.0f);   // -0 counts as 0
    return ((uint64_t)(u >> 31 ? ~u : u | 0x80000000u) << 32) | (0xFFFFFFFFu - token);
}
__device__ __forceinline__ float key_logit(uint64_t k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return __uint_as_float(u >> 31 ? u & 0x7FFFFFFFu : ~u);
}
__device__ __forceinline__ uint32_t key_token(uint64_t k) { return 0xFFFFFFFFu - (uint32_t)k; }
// order-preserving map of a finite double, never 0
__device__ __forceinline__ uint64_t score_key(double s) {
    const uint64_t u = (uint64_t)__double_as_longlong(s + 0.0);
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

__device__ __forceinline__ uint64_t umax64(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t umin64(uint64_t a, uint64_t b) { return a < b ? a : b; }

// the warp's 32 values in descending order of lane (bitonic network)
__device__ __forceinline__ uint64_t warp_sort(uint64_t v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int d = size >> 1; d; d >>= 1) {
            const uint64_t w = __shfl_xor_sync(0xffffffffu, v, d);
            const bool down = (lane & size) == 0, low = (lane & d) == 0;
            v = down == low ? umax64(v, w) : umin64(v, w);
        }
    return v;
}

// A value that at least k (<= 64) of the CTA's 256 values reach, near the k-th largest of them: of
// the 4 largest of each warp the k-th, beyond 32 the least of the warps' 8-th largest.
__device__ uint64_t block_threshold(uint64_t mine, int k, uint64_t* sh /* 32 */) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t v = warp_sort(mine);
    __syncthreads();                      // sh free
    if (k <= 32) {
        if (lane < 4) sh[warp * 4 + lane] = v;
    } else if (lane == 7) {
        sh[warp] = v;
    }
    __syncthreads();
    if (k <= 32) return __shfl_sync(0xffffffffu, warp_sort(sh[lane]), k - 1);
    uint64_t t = sh[0];
#pragma unroll
    for (int w = 1; w < BEAM_WARPS; w++) t = umin64(t, sh[w]);
    return t;
}

// list[0 .. n) -> its min(n, k) largest, sorted, in list[0 ..); all threads call it after a barrier
// that completed the list; ends with a barrier
__device__ int prune_keys(uint64_t* list, int n, int k, uint64_t* sh) {
    const int keep = n < k ? n : k;
    if (n <= BEAM_RANK) {                 // rank by counting: the keys are distinct
        const uint64_t mine = threadIdx.x < n ? list[threadIdx.x] : 0;
        int rank = 0;
        if (threadIdx.x < n)
            for (int i = 0; i < n; i++) rank += list[i] > mine;
        __syncthreads();
        if (threadIdx.x < n && rank < keep) list[rank] = mine;
        __syncthreads();
        return keep;
    }
    // long lists (an adverse order of the logits): one maximum after the other, each below the last
    uint64_t below = ~0ull;
    uint64_t found = 0;                   // thread r < keep remembers the r-th
    for (int r = 0; r < keep; r++) {
        uint64_t best = 0;
        for (int i = threadIdx.x; i < n; i += BEAM_THREADS) {
            const uint64_t x = list[i];
            if (x < below) best = umax64(best, x);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) best = umax64(best, __shfl_xor_sync(0xffffffffu, best, o));
        if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = best;
        __syncthreads();
        best = sh[0];
#pragma unroll
        for (int w = 1; w < BEAM_WARPS; w++) best = umax64(best, sh[w]);
        __syncthreads();
        below = best;
        if (threadIdx.x == r) found = best;
    }
    if (threadIdx.x < keep) list[threadIdx.x] = found;
    __syncthreads();
    return keep;
}

// tiles [begin(c), begin(c + 1)) belong to CTA c of G
__host__ __device__ __forceinline__ int64_t beam_begin(int64_t c, int64_t T, int64_t G) { return c * T / G; }
__device__ __forceinline__ int64_t beam_owner(int64_t u, int64_t T, int64_t G) { return ((u + 1) * G - 1) / T; }

struct BeamPart {
    double m, s;      // max (0 if there is none) and sum exp(x - m) of the part; s NaN: a NaN or +inf
};

__global__ void __launch_bounds__(BEAM_THREADS, BEAM_CTAS) beam_rows_kernel(
    const float* __restrict__ x, int64_t ld, int vocab, int k, int tpr, int64_t T, int max_parts,
    uint64_t* __restrict__ keys, BeamPart* __restrict__ parts) {
    __shared__ uint64_t list[BEAM_CAP];
    __shared__ uint64_t sh[32];
    __shared__ float wm[BEAM_WARPS];
    __shared__ double ws[BEAM_WARPS];
    __shared__ int count;
    pdl_wait();
    pdl_trigger();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int64_t G = gridDim.x, u0 = beam_begin(blockIdx.x, T, G), u1 = beam_begin(blockIdx.x + 1, T, G);
    float m = -INFINITY;
    double s = 0.0;
    int n = 0;                             // keys in the list after it was last pruned
    float tv = -INFINITY;                  // logits below (tv, ti) cannot be among the part's k largest
    uint32_t ti = 0;
    bool seeded = false;
    if (t == 0) count = 0;
    for (int64_t u = u0; u < u1; u++) {
        const int64_t row = u / tpr;
        const int base = (int)(u % tpr) * BEAM_TILE + t;
        const float* p = x + row * ld;
        float v[BEAM_PER];
#pragma unroll
        for (int j = 0; j < BEAM_PER; j++) {
            const int i = base + j * BEAM_THREADS;
            v[j] = i < vocab ? __ldcs(p + i) : -INFINITY;
        }
        // max and sum of exp: 16 terms in fp32, then on in 64 bits
        float mt = v[0];
#pragma unroll
        for (int j = 1; j < BEAM_PER; j++) mt = fmaxf(mt, v[j]);
        if (mt > m) {
            s *= (double)ex2((m - mt) * LOG2E);
            m = mt;
        }
        const float me = m == -INFINITY ? 0.0f : m;
        float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < BEAM_PER; j++) a[j & 3] += ex2((v[j] - me) * LOG2E);
        s += (double)((a[0] + a[1]) + (a[2] + a[3]));
        if (!seeded) {                     // the first tile of a part
            uint64_t best = 0;
            if (mt > -INFINITY) {
#pragma unroll
                for (int j = BEAM_PER - 1; j >= 0; j--)
                    if (v[j] == mt) best = beam_key(mt, (uint32_t)(base + j * BEAM_THREADS));
            }
            const uint64_t th = block_threshold(best, k, sh);
            tv = th ? key_logit(th) : -INFINITY;
            ti = key_token(th);
            seeded = true;
        }
        bool over = false;
        if (mt >= tv && mt > -INFINITY) {
#pragma unroll
            for (int j = 0; j < BEAM_PER; j++) {
                const uint32_t i = (uint32_t)(base + j * BEAM_THREADS);
                if (v[j] > tv || (v[j] == tv && i <= ti && v[j] > -INFINITY)) {
                    const int slot = atomicAdd(&count, 1);
                    list[slot] = beam_key(v[j], i);
                    over |= slot >= BEAM_LIMIT;
                }
            }
        }
        const bool last = u + 1 == u1 || (u + 1) % tpr == 0;
        // one barrier a tile; `count` is only read where every thread then waits before adding again
        if (__syncthreads_or(over || last)) {
            n = prune_keys(list, count, k, sh);
            if (t == 0) count = n;
            if (n == k) {
                tv = key_logit(list[k - 1]);
                ti = key_token(list[k - 1]);
            }
            __syncthreads();
        }
        if (last) {
            const int64_t part = blockIdx.x - beam_owner(row * tpr, T, G);
            uint64_t* out = keys + (row * max_parts + part) * k;
            if (t < k) out[t] = t < n ? list[t] : 0;
            // join the threads' sums at the CTA's maximum
            float M = m;
#pragma unroll
            for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
            if (lane == 0) wm[warp] = M;
            __syncthreads();
            M = wm[0];
#pragma unroll
            for (int w = 1; w < BEAM_WARPS; w++) M = fmaxf(M, wm[w]);
            if (M == -INFINITY) M = 0.0f;
            s *= (double)ex2((m - M) * LOG2E);
#pragma unroll
            for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            if (lane == 0) ws[warp] = s;
            if (t == 0) count = 0;
            __syncthreads();
            if (t == 0) {
                for (int w = 1; w < BEAM_WARPS; w++) s += ws[w];
                parts[row * max_parts + part] = {(double)M, s};
            }
            m = -INFINITY;
            s = 0.0;
            seeded = false;
        }
    }
}

struct Cand {
    double score;
    uint64_t key;
    int row;
};
__device__ __forceinline__ bool better(const Cand& a, const Cand& b) {
    return a.score > b.score || (a.score == b.score && (a.row < b.row || (a.row == b.row && a.key > b.key)));
}

constexpr int MERGE_PER = 4;
constexpr int MERGE_TILE = BEAM_THREADS * MERGE_PER;

// one CTA per group; candidate c = (rank c / lists in part-list c % lists): the heads come first
__global__ void __launch_bounds__(BEAM_THREADS) beam_merge_kernel(
    const uint64_t* __restrict__ keys, const BeamPart* __restrict__ parts, int tpr, int64_t T, int64_t G, int max_parts,
    const float* __restrict__ scores, const uint8_t* __restrict__ finished, int eos, int n_beams, int k,
    float* __restrict__ out_scores, int* __restrict__ out_rows, int* __restrict__ out_tokens) {
    __shared__ Cand list[BEAM_RANK + MERGE_TILE];
    __shared__ double lse[BEAM_MAX_BEAMS];
    __shared__ uint64_t sh[32];
    __shared__ Cand best_of[BEAM_WARPS];
    __shared__ int count;
    pdl_wait();
    pdl_trigger();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int64_t row0 = (int64_t)blockIdx.x * n_beams;
    // lse of each live beam; NaN: the beam offers no candidate; finished beams: 0 parts
    for (int b = warp; b < n_beams; b += BEAM_WARPS) {
        const int64_t row = row0 + b;
        const int np = (int)(beam_owner(row * tpr + tpr - 1, T, G) - beam_owner(row * tpr, T, G)) + 1;
        double M = -INFINITY;
        for (int i = lane; i < np; i += 32) {
            const BeamPart p = parts[row * max_parts + i];
            if (p.s > 0.0) M = fmax(M, p.m);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) M = fmax(M, __shfl_xor_sync(0xffffffffu, M, o));
        double s = 0.0;
        for (int i = lane; i < np; i += 32) {
            const BeamPart p = parts[row * max_parts + i];
            if (p.s != 0.0) s += p.s * exp(p.m - M);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) lse[b] = M + log(s);
    }
    if (t == 0) count = 0;
    __syncthreads();
    const int64_t lists = (int64_t)n_beams * max_parts, N = lists * k;
    int n = 0;
    bool full = false;                     // list[k - 1] bounds what may still enter
    Cand bound = {-INFINITY, 0, 0};
    for (int64_t c0 = 0; c0 < N; c0 += MERGE_TILE) {
        Cand v[MERGE_PER];
        uint64_t best = 0;
#pragma unroll
        for (int j = 0; j < MERGE_PER; j++) {
            const int64_t c = c0 + j * BEAM_THREADS + t;
            v[j] = {-INFINITY, 0, -1};
            if (c < N) {
                const int l = (int)(c % lists), rank = (int)(c / lists), b = l / max_parts, part = l % max_parts;
                const int64_t row = row0 + b;
                const double sc = scores[row];
                const bool done = finished && finished[row];
                if (done && rank == 0 && part == 0) {
                    v[j] = {sc, ~0ull, b};
                } else if (!done && part <= beam_owner(row * tpr + tpr - 1, T, G) - beam_owner(row * tpr, T, G)) {
                    const uint64_t key = keys[(row * max_parts + part) * k + rank];
                    if (key) v[j] = {sc + ((double)key_logit(key) - lse[b]), key, b};
                }
                if (!isfinite(sc) || !isfinite(v[j].score)) v[j].row = -1;
                if (v[j].row >= 0) best = umax64(best, score_key(v[j].score));
            }
        }
        const uint64_t th = c0 == 0 ? block_threshold(best, k, sh) : 0;
        bool over = false;
#pragma unroll
        for (int j = 0; j < MERGE_PER; j++)
            if (v[j].row >= 0 && (full ? better(v[j], bound) : score_key(v[j].score) >= th)) {
                const int slot = atomicAdd(&count, 1);
                list[slot] = v[j];
                over |= slot >= BEAM_RANK;
            }
        if (__syncthreads_or(over || c0 + MERGE_TILE >= N)) {
            n = count;
            const int keep = n < k ? n : k;
            if (n <= BEAM_RANK) {
                Cand mine = {0, 0, 0};
                int rank = 0;
                if (t < n) {
                    mine = list[t];
                    for (int i = 0; i < n; i++) rank += better(list[i], mine);
                }
                __syncthreads();
                if (t < n && rank < keep) list[rank] = mine;
            } else {
                Cand found = {0, 0, 0}, below = {INFINITY, 0, 0};
                for (int r = 0; r < keep; r++) {
                    Cand b = {-INFINITY, 0, INT32_MAX};
                    for (int i = t; i < n; i += BEAM_THREADS) {
                        const Cand x = list[i];
                        if (better(below, x) && better(x, b)) b = x;
                    }
#pragma unroll
                    for (int o = 16; o; o >>= 1) {
                        Cand w;
                        w.score = __shfl_xor_sync(0xffffffffu, b.score, o);
                        w.key = __shfl_xor_sync(0xffffffffu, b.key, o);
                        w.row = __shfl_xor_sync(0xffffffffu, b.row, o);
                        if (better(w, b)) b = w;
                    }
                    if (lane == 0) best_of[warp] = b;
                    __syncthreads();
                    b = best_of[0];
#pragma unroll
                    for (int w = 1; w < BEAM_WARPS; w++)
                        if (better(best_of[w], b)) b = best_of[w];
                    __syncthreads();
                    below = b;
                    if (t == r) found = b;
                }
                if (t < keep) list[t] = found;
            }
            __syncthreads();
            n = keep;
            if (t == 0) count = n;
            __syncthreads();
            full = n == k;
            if (full) bound = list[k - 1];
        }
    }
    if (t < k) {
        const int64_t o = (int64_t)blockIdx.x * k + t;
        const bool none = t >= n;
        const Cand c = none ? Cand{-INFINITY, 0, 0} : list[t];
        out_scores[o] = (float)c.score;
        out_rows[o] = none ? -1 : (int)(row0 + c.row);
        out_tokens[o] = none ? -1 : (c.key == ~0ull ? eos : (int)key_token(c.key));
    }
}

struct BeamPlan {
    int tpr, max_parts;
    int64_t T, G;
    size_t keys_bytes, bytes;
};
// Ranges of whole tiles, as equal as whole tiles allow: with fewer than BEAM_CTAS CTAs per SM's worth
// of tiles one each, else the least number of tiles per CTA that one wave of CTAs can take.
static BeamPlan beam_plan(int n_groups, int n_beams, int64_t vocab, int k) {
    BeamPlan p;
    const int64_t rows = (int64_t)n_groups * n_beams;
    p.tpr = (int)((vocab + BEAM_TILE - 1) / BEAM_TILE);
    p.T = rows * p.tpr;
    const int64_t wave = (int64_t)BEAM_CTAS * num_sms();
    const int64_t per = (p.T + wave - 1) / wave;
    p.G = (p.T + per - 1) / per;
    const int64_t least = p.T / p.G;                      // tiles of the shortest range
    p.max_parts = (int)((p.tpr + least - 1) / least + 1);
    if (p.max_parts > p.tpr) p.max_parts = p.tpr;
    p.keys_bytes = align256((size_t)rows * p.max_parts * k * 8);
    p.bytes = p.keys_bytes + align256((size_t)rows * p.max_parts * sizeof(BeamPart));
    return p;
}

size_t beam_scratch_bytes(int n_groups, int n_beams, int64_t vocab, int k) {
    return beam_plan(n_groups, n_beams, vocab, k).bytes;
}

cudaError_t launch_beam_select(const float* logits, int64_t ld, int n_groups, int n_beams, int64_t vocab,
                               const float* scores, const uint8_t* finished, int eos, int k, float* out_scores,
                               int* out_rows, int* out_tokens, void* scratch, cudaStream_t st) {
    const BeamPlan p = beam_plan(n_groups, n_beams, vocab, k);
    uint64_t* keys = (uint64_t*)scratch;
    BeamPart* parts = (BeamPart*)((uint8_t*)scratch + p.keys_bytes);
    cudaError_t e = launch_pdl(beam_rows_kernel, dim3((unsigned)p.G), dim3(BEAM_THREADS), 0, st, logits, ld, (int)vocab, k,
                               p.tpr, p.T, p.max_parts, keys, parts);
    if (e != cudaSuccess) return e;
    return launch_pdl(beam_merge_kernel, dim3((unsigned)n_groups), dim3(BEAM_THREADS), 0, st, (const uint64_t*)keys,
                      (const BeamPart*)parts, p.tpr, p.T, p.G, p.max_parts, scores, finished, eos, n_beams, k, out_scores,
                      out_rows, out_tokens);
}

}  // namespace dcg
