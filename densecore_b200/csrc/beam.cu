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
// logits, and per tile and warp the max and the sum of exp(x - max) over the others: sums that do not
// depend on how the rows were cut, so that rows with the same logits tie exactly.  beam_merge_kernel, one CTA per group, joins them.
// What bounds it: HBM in the pass over many rows (512 beams of 128,256 logits: 69 us with the merge's
// 11, 4.5 TB/s in the pass), the two launches' latency over few (4 beams of 151,936: 9.5 us).
#include <math.h>

#include "../../include/dcgpu.h"
#include "common.cuh"
#include "kernels.h"

namespace dcg {

constexpr int BEAM_THREADS = 256;
constexpr int BEAM_WARPS = BEAM_THREADS / 32;
constexpr int BEAM_PER = 16;                             // logits per thread and tile
constexpr int BEAM_TILE = BEAM_THREADS * BEAM_PER;
constexpr int BEAM_CTAS = 4;                             // resident CTAs per SM (36 KB of keys each): 512 beams 70 us, with 3 76, with 2 85
constexpr int BEAM_RANK = 256;                           // lists up to this long are sorted by counting
constexpr int BEAM_FEW = 64;                             // longer ones after a threshold
constexpr int BEAM_CAP = 2 * BEAM_MAX_K + 32 + BEAM_TILE;   // pruned beyond 2 k + 32: a whole tile always fits
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float warp_max(float x) {
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));   // NaN only if all are
    return y;
}
// (x0, x1) * a + b, and sums, two at a time
__device__ __forceinline__ uint64_t pack2(float x0, float x1) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x0), "f"(x1));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t r, float& x0, float& x1) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x0), "=f"(x1) : "l"(r)); }
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t a, uint64_t b) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
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
__device__ __forceinline__ uint64_t umax64(uint64_t a, uint64_t b) { return a > b ? a : b; }

// order-preserving map of a float (NaN apart), never 0
__device__ __forceinline__ uint32_t float_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u >> 31 ? ~u : u | 0x80000000u;
}

// the warp's 32 values in descending order of lane (bitonic network)
__device__ __forceinline__ uint32_t warp_sort(uint32_t v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int d = size >> 1; d; d >>= 1) {
            const uint32_t w = __shfl_xor_sync(0xffffffffu, v, d);
            v = ((lane & size) == 0) == ((lane & d) == 0) ? max(v, w) : min(v, w);
        }
    return v;
}

// A value that at least k (<= 64) of the CTA's 256 values reach, near the k-th largest of them: the
// k-th of the warps' 4 (k > 16: 8) largest.  sh[64]: where warp 0 finds them; the result is left in
// sh[0].  Starts and ends with a barrier.
__device__ uint32_t block_threshold(uint32_t mine, int k, uint32_t* sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int each = k <= 16 ? 4 : 8;
    const uint32_t v = warp_sort(mine);
    __syncthreads();                      // sh free
    if (lane < each) sh[warp * each + lane] = v;
    __syncthreads();
    if (warp == 0) {
        uint32_t a = warp_sort(sh[lane]);
        if (each == 8) {
            // two sorted halves, one of them reversed: their maxima are the 32 largest, their minima the rest
            const uint32_t b = __shfl_xor_sync(0xffffffffu, warp_sort(sh[32 + lane]), 31);
            a = warp_sort(k <= 32 ? max(a, b) : min(a, b));
        }
        a = __shfl_sync(0xffffffffu, a, (k - 1) & 31);
        if (lane == 0) sh[0] = a;
    }
    __syncthreads();
    return sh[0];
}

// shared memory of the selection
struct Select {
    uint32_t sh[64];
    uint64_t top[BEAM_WARPS];
    int count;                            // of the growing list
    int kept;                             // of the list that a pruning makes
};

// list[0 .. n) -> its min(n, k) largest, sorted, in list[0 ..); tmp[BEAM_RANK]: room of its own.
// All threads call it after a barrier that completed the list; ends with a barrier.
__device__ int prune_keys(uint64_t* list, uint64_t* tmp, int n, int k, Select& S) {
    const int keep = n < k ? n : k;
    int m = n;
    const uint64_t* from = list;
    if (n > BEAM_FEW) {                   // first those that reach a threshold, from each thread's largest
        uint32_t best = 0;
        for (int i = threadIdx.x; i < n; i += BEAM_THREADS) best = max(best, (uint32_t)(list[i] >> 32));
        if (threadIdx.x == 0) S.kept = 0;
        const uint32_t th = block_threshold(best, k, S.sh);
        for (int i = threadIdx.x; i < n; i += BEAM_THREADS) {
            const uint64_t x = list[i];
            if ((uint32_t)(x >> 32) >= th) {
                const int slot = atomicAdd(&S.kept, 1);
                if (slot < BEAM_RANK) tmp[slot] = x;
            }
        }
        __syncthreads();
        m = S.kept;
        from = tmp;
    }
    if (m <= BEAM_RANK) {                 // rank by counting: the keys are distinct
        const uint64_t mine = threadIdx.x < m ? from[threadIdx.x] : 0;
        int rank = 0;
        if (threadIdx.x < m)
#pragma unroll 4
            for (int i = 0; i < m; i++) rank += from[i] > mine;
        __syncthreads();
        if (threadIdx.x < m && rank < keep) list[rank] = mine;
        __syncthreads();
        return keep;
    }
    // many equal logits: one maximum after the other, each below the last
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
        if ((threadIdx.x & 31) == 0) S.top[threadIdx.x >> 5] = best;
        __syncthreads();
        best = S.top[0];
#pragma unroll
        for (int w = 1; w < BEAM_WARPS; w++) best = umax64(best, S.top[w]);
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

// a tile of a row: logits base, base + 256, ... below vocab, -inf beyond
__device__ __forceinline__ void load_tile(float (&v)[BEAM_PER], const float* __restrict__ p, int base, int vocab, bool whole) {
    if (whole) {
#pragma unroll
        for (int j = 0; j < BEAM_PER; j++) v[j] = __ldcs(p + base + j * BEAM_THREADS);
    } else {
#pragma unroll
        for (int j = 0; j < BEAM_PER; j++) {
            const int i = base + j * BEAM_THREADS;
            v[j] = i < vocab ? __ldcs(p + i) : -INFINITY;
        }
    }
}

// One part of a row: tiles u0 .. u1 - 1 of the whole, all of row `row`.  The list takes the logits
// that reach (tv, ti).  The first tile sets the threshold, at its r-th largest logit:
//   CHECKED = false: r may be below k when the part is long (about 4 k logits of the part are then
//     expected to reach it), and no thread waits for another until the part is read.  Returns false
//     if fewer than k logits came, or more than the list holds.
//   CHECKED = true: r = k, which at least k logits reach whatever the order of the logits; the list
//     is pruned, and the threshold raised, whenever it has grown.
template <bool CHECKED>
__device__ bool read_part(const float* __restrict__ p, int64_t u0, int64_t u1, int tile0, int vocab, int k, int tpr,
                          float2* __restrict__ sums, uint64_t* list, uint64_t* tmp, Select& S) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int tiles = (int)(u1 - u0);
    const int r = CHECKED ? k : min(k, max(8, (4 * k + tiles - 1) / tiles));
    float tv = -INFINITY;
    uint32_t ti = 0xFFFFFFFFu;
    if (t == 0) S.count = 0;
    float next[BEAM_PER];
    load_tile(next, p, tile0 * BEAM_TILE + t, vocab, tile0 + 1 < tpr);
    for (int i = 0; i < tiles; i++) {
        const int base = (tile0 + i) * BEAM_TILE + t;
        float v[BEAM_PER];
#pragma unroll
        for (int j = 0; j < BEAM_PER; j++) v[j] = next[j];
        if (i + 1 < tiles) load_tile(next, p, base + BEAM_TILE, vocab, tile0 + i + 2 < tpr);
        float m4[4];
#pragma unroll
        for (int j = 0; j < 4; j++) m4[j] = fmaxf(fmaxf(v[j], v[j + 4]), fmaxf(v[j + 8], v[j + 12]));
        const float mt = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        const float mw = warp_max(mt);
        const float me = mw == -INFINITY ? 0.0f : mw;
        // s = sum 2^(v c - me c), c = log2 e in fp32, as fma(v, c, -h) with h = me c rounded; what that
        // rounding lost is one factor for the whole warp
        const float h = me * LOG2E, l = fmaf(me, LOG2E, -h);
        const uint64_t c2 = pack2(LOG2E, LOG2E), h2 = pack2(-h, -h);
        uint64_t a0 = 0, a1 = 0;
#pragma unroll
        for (int j = 0; j < BEAM_PER; j += 4) {
            float e0, e1, e2, e3;
            unpack2(fma2(pack2(v[j], v[j + 1]), c2, h2), e0, e1);
            unpack2(fma2(pack2(v[j + 2], v[j + 3]), c2, h2), e2, e3);
            a0 = add2(a0, pack2(ex2(e0), ex2(e1)));
            a1 = add2(a1, pack2(ex2(e2), ex2(e3)));
        }
        float s, s1;
        unpack2(add2(a0, a1), s, s1);
        s = (s + s1) * ex2(-l);
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        float r1 = s - 1.0f;               // the sum without the largest logit's own 1
        if (!(s >= 1.015625f && fabsf(me) < 16777216.0f)) {
            // one logit far above the rest (lse - max would be lost next to 1), or me so large that l, up to half a
            // step of h (1 at |me| = 2^24, beyond 126 from 5 x 10^9 on), takes the two factors out of fp32's range:
            // the rest alone, from v - me.  +inf makes it NaN, as a NaN does
            bool skip = lane == __ffs(__ballot_sync(0xffffffffu, mt == mw)) - 1;
            r1 = me == INFINITY ? NAN : 0.0f;
#pragma unroll
            for (int j = 0; j < BEAM_PER; j++) {
                if (skip && v[j] == mw) skip = false;
                else r1 += ex2((v[j] - me) * LOG2E);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) r1 += __shfl_xor_sync(0xffffffffu, r1, o);
        }
        if (lane == 0) sums[(u0 + i) * BEAM_WARPS + warp] = make_float2(mw, r1);
        if (i == 0) tv = key_logit((uint64_t)block_threshold(float_key(mt), r, S.sh) << 32);
        bool over = false;
        if (mw >= tv && mw > -INFINITY) {
#pragma unroll
            for (int g = 0; g < 4; g++) {
                if (!__any_sync(0xffffffffu, m4[g] >= tv)) continue;
#pragma unroll
                for (int j = g; j < BEAM_PER; j += 4) {
                    const uint32_t at = (uint32_t)(base + j * BEAM_THREADS);
                    if (v[j] > tv || (v[j] == tv && at <= ti && v[j] > -INFINITY)) {
                        const int slot = atomicAdd(&S.count, 1);
                        if (CHECKED || slot < BEAM_CAP) list[slot] = beam_key(v[j], at);
                        if (CHECKED) over |= slot >= 2 * k + 32;
                    }
                }
            }
        }
        // the count is only read where every thread then waits before adding again
        if (CHECKED && __syncthreads_or(over)) {
            const int n = prune_keys(list, tmp, S.count, k, S);
            if (t == 0) S.count = n;
            if (n == k) {
                tv = key_logit(list[k - 1]);
                ti = key_token(list[k - 1]);
            }
            __syncthreads();
        }
    }
    __syncthreads();
    return S.count <= BEAM_CAP && (S.count >= k || r == k);
}

__global__ void __launch_bounds__(BEAM_THREADS, BEAM_CTAS) beam_rows_kernel(
    const float* __restrict__ x, int64_t ld, int vocab, int k, int tpr, int64_t T, int max_parts,
    uint64_t* __restrict__ keys, float2* __restrict__ sums) {
    __shared__ uint64_t list[BEAM_CAP];
    __shared__ uint64_t tmp[BEAM_RANK];
    __shared__ Select S;
    pdl_wait();
    pdl_trigger();
    const int64_t G = gridDim.x, end = beam_begin(blockIdx.x + 1, T, G);
    for (int64_t u0 = beam_begin(blockIdx.x, T, G), u1; u0 < end; u0 = u1) {
        const int64_t row = u0 / tpr;
        const int tile0 = (int)(u0 % tpr);
        u1 = u0 + tpr - tile0 < end ? u0 + tpr - tile0 : end;
        const float* p = x + row * ld;
        if (!read_part<false>(p, u0, u1, tile0, vocab, k, tpr, sums, list, tmp, S)) {
            __syncthreads();
            read_part<true>(p, u0, u1, tile0, vocab, k, tpr, sums, list, tmp, S);
        }
        const int n = prune_keys(list, tmp, S.count, k, S);
        const int64_t part = blockIdx.x - beam_owner(row * tpr, T, G);
        if (threadIdx.x < k) keys[(row * max_parts + part) * k + threadIdx.x] = threadIdx.x < n ? list[threadIdx.x] : 0;
        __syncthreads();
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
constexpr int MERGE_SUMS = 8;                            // a thread's tile sums under way (35 beams: 16.8 us, with 4 or 6 17.1, with 16 19)
constexpr int MERGE_TILE = BEAM_THREADS * MERGE_PER;

// one CTA per group; candidate c = (rank c / lists in part-list c % lists): the heads come first.  (One CTA per SM
// in the bounds and rolled loops: held to 64 registers, it spilled and took 2 us more.)
__global__ void __launch_bounds__(BEAM_THREADS, 1) beam_merge_kernel(
    const uint64_t* __restrict__ keys, const float2* __restrict__ sums, int tpr, int64_t T, int G, int max_parts,
    const float* __restrict__ scores, const uint8_t* __restrict__ finished, int eos, int n_beams, int k,
    float* __restrict__ out_scores, int* __restrict__ out_rows, int* __restrict__ out_tokens) {
    __shared__ Cand list[BEAM_RANK + MERGE_TILE];
    __shared__ double score_of[BEAM_MAX_BEAMS], lse_of[BEAM_MAX_BEAMS];   // not finite: no candidate
    __shared__ int n_parts[BEAM_MAX_BEAMS];     // of each beam; 0: finished
    __shared__ Cand tmp[BEAM_RANK];
    __shared__ Select S;
    __shared__ Cand best_of[BEAM_WARPS];
    pdl_wait();
    pdl_trigger();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int64_t row0 = (int64_t)blockIdx.x * n_beams;
    const int lists = n_beams * max_parts, N = lists * k;   // max_parts <= G: below 2^31
#pragma unroll 1
    for (int b = t; b < n_beams; b += BEAM_THREADS) {
        const int64_t u = (row0 + b) * tpr;
        n_parts[b] = finished && finished[row0 + b] ? 0 : (int)(beam_owner(u + tpr - 1, T, G) - beam_owner(u, T, G)) + 1;
    }
#pragma unroll 1
    for (int b = warp; b < n_beams; b += BEAM_WARPS) {
        const float2* p = sums + (row0 + b) * tpr * BEAM_WARPS;
        const int np = tpr * BEAM_WARPS;
        float M = -INFINITY;
        double s = 0.0;
#pragma unroll 1
        for (int i0 = 0; i0 < np; i0 += 32 * MERGE_SUMS) {
            float2 q[MERGE_SUMS];                 // loaded once
#pragma unroll
            for (int i = 0; i < MERGE_SUMS; i++) {
                const int at = i0 + 32 * i + lane;
                q[i] = at < np ? p[at] : make_float2(-INFINITY, 0.0f);
            }
            float m = q[0].x;
#pragma unroll
            for (int i = 1; i < MERGE_SUMS; i++) m = fmaxf(m, q[i].x);
            m = warp_max(m);
            if (m > M) {
                s *= (double)ex2((M - m) * LOG2E);
                M = m;
            }
#pragma unroll
            for (int i = 0; i < MERGE_SUMS; i++)
                if (q[i].x > -INFINITY || q[i].y != 0.0f) s += (1.0 + (double)q[i].y) * (double)ex2((q[i].x - M) * LOG2E);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) {
            score_of[b] = scores[row0 + b];
            lse_of[b] = (double)M + log(s);
        }
    }
    if (t == 0) S.count = 0;
    __syncthreads();
    int n = 0;
    bool full = false;                     // list[k - 1] bounds what may still enter
    Cand bound = {-INFINITY, 0, 0};
    uint32_t th = 0;
    int quiet = 0;                         // candidates since the last that came in
#pragma unroll 1
    for (int c0 = 0; c0 < N && quiet < lists; c0 += MERGE_TILE) {
        Cand v[MERGE_PER];
        uint32_t best = 0;
#pragma unroll
        for (int j = 0; j < MERGE_PER; j++) {
            const int c = c0 + j * BEAM_THREADS + t;
            v[j] = {-INFINITY, 0, -1};
            if (c < N) {
                const int rank = c / lists, l = c - rank * lists, b = l / max_parts, part = l - b * max_parts;
                if (n_parts[b] == 0 ? rank == 0 && part == 0 : part < n_parts[b]) {
                    const uint64_t key = n_parts[b] == 0 ? ~0ull : keys[((row0 + b) * max_parts + part) * k + rank];
                    const double score = n_parts[b] == 0 ? score_of[b] : score_of[b] + ((double)key_logit(key) - lse_of[b]);
                    if (key && isfinite(score)) {
                        v[j] = {score, key, b};
                        best = max(best, float_key(__double2float_rd(score)));
                    }
                }
            }
        }
        // scores rounded down keep their order
        if (c0 == 0) th = block_threshold(best, k, S.sh);
        bool over = false, came = false;
#pragma unroll
        for (int j = 0; j < MERGE_PER; j++)
            if (v[j].row >= 0 && (full ? better(v[j], bound) : float_key(__double2float_rd(v[j].score)) >= th)) {
                const int slot = atomicAdd(&S.count, 1);
                list[slot] = v[j];
                over |= slot >= BEAM_RANK;
                came = true;
            }
        // the lists descend: once none of a whole rank comes in, nothing behind does (16 beams of 119,088 logits
        // in one group, k 32: 48 us without this)
        bool last = c0 + MERGE_TILE >= N;
        if (!last) {
            quiet = __syncthreads_or(came) ? 0 : quiet + MERGE_TILE;
            last = quiet >= lists;
        }
        if (__syncthreads_or(over || last)) {
            n = S.count;
            const int keep = n < k ? n : k;
            int m = n;
            const Cand* from = list;
            if (n > BEAM_FEW) {            // as prune_keys, by score alone
                uint32_t top = 0;
#pragma unroll 1
                for (int i = t; i < n; i += BEAM_THREADS) top = max(top, float_key(__double2float_rd(list[i].score)));
                if (t == 0) S.kept = 0;
                const uint32_t reach = block_threshold(top, k, S.sh);
#pragma unroll 1
                for (int i = t; i < n; i += BEAM_THREADS)
                    if (float_key(__double2float_rd(list[i].score)) >= reach) {
                        const int slot = atomicAdd(&S.kept, 1);
                        if (slot < BEAM_RANK) tmp[slot] = list[i];
                    }
                __syncthreads();
                m = S.kept;
                from = tmp;
            }
            if (m <= BEAM_RANK) {
                Cand mine = {0, 0, 0};
                int rank = 0;
                if (t < m) {
                    mine = from[t];
#pragma unroll 4
                    for (int i = 0; i < m; i++) rank += better(from[i], mine);
                }
                __syncthreads();
                if (t < m && rank < keep) list[rank] = mine;
            } else {
                Cand found = {0, 0, 0}, below = {INFINITY, 0, 0};
#pragma unroll 1
                for (int r = 0; r < keep; r++) {
                    Cand b = {-INFINITY, 0, INT32_MAX};
#pragma unroll 1
                    for (int i = t; i < n; i += BEAM_THREADS) {
                        const Cand x = list[i];
                        if (better(below, x) && better(x, b)) b = x;
                    }
#pragma unroll 1
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
#pragma unroll 1
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
            if (t == 0) S.count = n;
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
    p.bytes = p.keys_bytes + align256((size_t)p.T * BEAM_WARPS * sizeof(float2));
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
    float2* sums = (float2*)((uint8_t*)scratch + p.keys_bytes);
    cudaError_t e = launch_pdl(beam_rows_kernel, dim3((unsigned)p.G), dim3(BEAM_THREADS), 0, st, logits, ld, (int)vocab, k,
                               p.tpr, p.T, p.max_parts, keys, sums);
    if (e != cudaSuccess) return e;
    return launch_pdl(beam_merge_kernel, dim3((unsigned)n_groups), dim3(BEAM_THREADS), 0, st, (const uint64_t*)keys,
                      (const float2*)sums, p.tpr, p.T, (int)p.G, p.max_parts, scores, finished, eos, n_beams, k, out_scores,
                      out_rows, out_tokens);
}

}  // namespace dcg
