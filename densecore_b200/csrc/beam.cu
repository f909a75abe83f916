// beam.cu -- beam search's selection: log-softmax of every beam's logits, added to the beam's score,
// and the k best (beam, token) pairs of each group of beams.
//
// The reference samples one token per sequence on the host (core/src/inference.cpp:2127-2244).
// Candidate (b, t) scores s_b + (x_bt - lse_b), lse_b = log sum_t exp x_bt.  Within a
// beam the order of the candidates is that of the logits (exact: no rounding decides it), so each
// beam contributes at most its k largest logits; across beams the scores are compared in 64 bits.
#include <math.h>

#include "../../include/dcgpu.h"
#include "common.cuh"
#include "kernels.h"

namespace dcg {

constexpr int BEAM_THREADS = 256;

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

__device__ uint64_t block_max_key(uint64_t v, uint64_t* sh) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const uint64_t w = __shfl_xor_sync(0xffffffffu, v, o);
        v = w > v ? w : v;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh[0];
    for (int w = 1; w < BEAM_THREADS / 32; w++) v = sh[w] > v ? sh[w] : v;
    return v;
}

// one CTA per row: lse in 64 bits, then the k largest keys one by one
__global__ void __launch_bounds__(BEAM_THREADS) beam_rows_kernel(const float* __restrict__ x, int64_t ld, int64_t vocab,
                                                                 int k, uint64_t* __restrict__ keys, double* __restrict__ lse) {
    __shared__ uint64_t sh[BEAM_THREADS / 32];
    __shared__ double sums[BEAM_THREADS / 32];
    pdl_wait();
    pdl_trigger();
    const float* row = x + (int64_t)blockIdx.x * ld;
    uint64_t best = 0;
    for (int64_t i = threadIdx.x; i < vocab; i += BEAM_THREADS) {
        const float v = row[i];
        const uint64_t key = v > -INFINITY ? beam_key(v, (uint32_t)i) : 0;
        best = key > best ? key : best;
    }
    best = block_max_key(best, sh);
    const float m = best ? key_logit(best) : 0.0f;
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < vocab; i += BEAM_THREADS) s += (double)expf(row[i] - m);
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < BEAM_THREADS / 32; w++) s += sums[w];
        lse[blockIdx.x] = (double)m + log(s);
    }
    for (int r = 0; r < k; r++) {
        if (threadIdx.x == 0) keys[(int64_t)blockIdx.x * k + r] = best;
        uint64_t next = 0;
        for (int64_t i = threadIdx.x; i < vocab; i += BEAM_THREADS) {
            const float v = row[i];
            const uint64_t key = v > -INFINITY ? beam_key(v, (uint32_t)i) : 0;
            if (key < best && key > next) next = key;
        }
        best = block_max_key(next, sh);
    }
}

struct Cand {
    double score;
    uint64_t order;   // row within the group ascending, then the row's own order (its rank)
};
__device__ __forceinline__ bool better(const Cand& a, const Cand& b) {
    return a.score > b.score || (a.score == b.score && a.order < b.order);
}

// one CTA per group: the k best of its beams' candidates, one by one
__global__ void __launch_bounds__(BEAM_THREADS) beam_merge_kernel(
    const uint64_t* __restrict__ keys, const double* __restrict__ lse, const float* __restrict__ scores,
    const uint8_t* __restrict__ finished, int eos, int n_beams, int k, float* __restrict__ out_scores,
    int* __restrict__ out_rows, int* __restrict__ out_tokens) {
    __shared__ Cand sh[BEAM_THREADS / 32];
    pdl_wait();
    pdl_trigger();
    const int row0 = blockIdx.x * n_beams, n = n_beams * k;
    Cand last = {INFINITY, 0};
    bool first = true;
    for (int r = 0; r < k; r++) {
        Cand best = {-INFINITY, ~0ull};
        for (int c = threadIdx.x; c < n; c += BEAM_THREADS) {
            const int row = row0 + c / k;
            const double s = scores[row], l = lse[row];
            Cand x = {-INFINITY, (uint64_t)c};
            if (!isfinite(s)) continue;
            if (finished && finished[row]) {
                if (c % k) continue;
                x.score = s;
            } else {
                const uint64_t key = keys[(int64_t)row * k + c % k];
                if (!key || !isfinite(l)) continue;
                x.score = s + ((double)key_logit(key) - l);
            }
            if ((first || better(last, x)) && better(x, best)) best = x;
        }
        for (int o = 16; o; o >>= 1) {
            Cand w;
            w.score = __shfl_xor_sync(0xffffffffu, best.score, o);
            w.order = __shfl_xor_sync(0xffffffffu, best.order, o);
            if (better(w, best)) best = w;
        }
        __syncthreads();
        if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = best;
        __syncthreads();
        best = sh[0];
        for (int w = 1; w < BEAM_THREADS / 32; w++)
            if (better(sh[w], best)) best = sh[w];
        if (threadIdx.x == 0) {
            const int64_t o = (int64_t)blockIdx.x * k + r;
            const bool none = best.order == ~0ull;
            const int row = none ? -1 : row0 + (int)(best.order / k);
            out_scores[o] = none ? -INFINITY : (float)best.score;
            out_rows[o] = row;
            out_tokens[o] = none ? -1 : (finished && finished[row] ? eos : (int)key_token(keys[(int64_t)row * k + best.order % k]));
        }
        last = best;
        first = false;
        if (best.order == ~0ull) last = {-INFINITY, ~0ull};
    }
}

size_t beam_scratch_bytes(int n_groups, int n_beams, int64_t vocab, int k) {
    const size_t rows = (size_t)n_groups * n_beams;
    return align256(rows * k * 8) + align256(rows * 8);
}

cudaError_t launch_beam_select(const float* logits, int64_t ld, int n_groups, int n_beams, int64_t vocab,
                               const float* scores, const uint8_t* finished, int eos, int k, float* out_scores,
                               int* out_rows, int* out_tokens, void* scratch, cudaStream_t st) {
    const size_t rows = (size_t)n_groups * n_beams;
    uint64_t* keys = (uint64_t*)scratch;
    double* lse = (double*)((uint8_t*)scratch + align256(rows * k * 8));
    cudaError_t e = launch_pdl(beam_rows_kernel, dim3((unsigned)rows), dim3(BEAM_THREADS), 0, st, logits, ld, vocab, k, keys, lse);
    if (e != cudaSuccess) return e;
    return launch_pdl(beam_merge_kernel, dim3((unsigned)n_groups), dim3(BEAM_THREADS), 0, st, (const uint64_t*)keys,
                      (const double*)lse, scores, finished, eos, n_beams, k, out_scores, out_rows, out_tokens);
}

}  // namespace dcg
