// attn_tree.cu -- attention of a drafted token tree over DenseCore's paged fp16 KV cache.
//
// Beside the causal masks of the reference's attention selector (core/src/inference.cpp:1506-1573):
// drafted token i sees the whole history and, of the draft, the tokens
// whose bit is set in its mask row (its ancestors and itself).  Layout and checks as attn.cu.
#include <math.h>

#include "../../include/dcgpu.h"
#include "common.cuh"
#include "kernels.h"

namespace dcg {

constexpr int HD = 128;
constexpr int KVB = 16;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int TREE_WARPS = 8;

__device__ int g_tree_error = 0;

cudaError_t tree_device_error(int* out, bool clear) {
    cudaError_t e = cudaMemcpyFromSymbol(out, g_tree_error, sizeof(int));
    if (e == cudaSuccess && clear && *out) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_tree_error, &zero, sizeof(int));
    }
    return e;
}

// one CTA per (drafted token, query head); warp w takes keys w, w + 8, ...; a lane holds 4 dims
__global__ void __launch_bounds__(TREE_WARPS * 32) tree_simple_kernel(
    const float* __restrict__ q, const __half* __restrict__ karena, const __half* __restrict__ varena,
    int64_t n_arena_blocks, int n_layer, int layer, const int* __restrict__ bt, int mbs,
    const int* __restrict__ seq_starts, const int* __restrict__ ctx, const int64_t* __restrict__ mask,
    int words, int n_tok, int max_seq_tokens, int hq, int hkv, float scale_log2, float* __restrict__ out) {
    __shared__ float wm[TREE_WARPS], wl[TREE_WARPS], wo[TREE_WARPS][HD];
    pdl_wait();
    pdl_trigger();
    const int seq = blockIdx.y, i = blockIdx.x, h = blockIdx.z;
    const int s0 = seq_starts[seq], s1 = seq_starts[seq + 1], ns = s1 - s0, L = ctx[seq];
    if (s0 < 0 || s1 < s0 || s1 > n_tok || ns > max_seq_tokens || L < ns || L > mbs * KVB || ns > 64 * words) {
        if (threadIdx.x == 0) atomicExch(&g_tree_error, DCG_DEVERR_INDEX);
        return;
    }
    if (i >= ns) return;
    const int hist = L - ns, kvh = h / (hq / hkv);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t at = ((int64_t)(s0 + i) * hq + h) * HD + 4 * lane;
    const float4 qv = *(const float4*)(q + at);
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j = warp; j < L; j += TREE_WARPS) {
        const int t = j - hist;
        if (t >= 0 && !((mask[(int64_t)(s0 + i) * words + t / 64] >> (t % 64)) & 1)) continue;
        const int page = bt[(int64_t)seq * mbs + j / KVB];
        const bool there = page >= 0 && page < n_arena_blocks;
        if (!there) atomicExch(&g_tree_error, DCG_DEVERR_INDEX);
        const int64_t slot = (((int64_t)page * n_layer + layer) * KVB + j % KVB) * hkv + kvh;
        uint2 kw = make_uint2(0, 0), vw = kw;
        if (there) {
            kw = *(const uint2*)(karena + slot * HD + 4 * lane);
            vw = *(const uint2*)(varena + slot * HD + 4 * lane);
        }
        const float2 k0 = __half22float2(*(const __half2*)&kw.x), k1 = __half22float2(*(const __half2*)&kw.y);
        const float2 v0 = __half22float2(*(const __half2*)&vw.x), v1 = __half22float2(*(const __half2*)&vw.y);
        float s = qv.x * k0.x + qv.y * k0.y + qv.z * k1.x + qv.w * k1.y;
#pragma unroll
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        s *= scale_log2;
        const float mn = fmaxf(m, s), c = m == -INFINITY ? 0.0f : exp2f(m - mn), p = exp2f(s - mn);
        m = mn;
        l = l * c + p;
        o.x = o.x * c + p * v0.x;
        o.y = o.y * c + p * v0.y;
        o.z = o.z * c + p * v1.x;
        o.w = o.w * c + p * v1.y;
    }
    if (lane == 0) { wm[warp] = m; wl[warp] = l; }
    *(float4*)&wo[warp][4 * lane] = o;
    __syncthreads();
    if (threadIdx.x < HD) {
        float M = -INFINITY, Ls = 0.0f, O = 0.0f;
        for (int w = 0; w < TREE_WARPS; w++)
            if (wl[w] != 0.0f) M = fmaxf(M, wm[w]);
        for (int w = 0; w < TREE_WARPS; w++)
            if (wl[w] != 0.0f) {
                const float f = exp2f(wm[w] - M);
                Ls += wl[w] * f;
                O += wo[w][threadIdx.x] * f;
            }
        out[((int64_t)(s0 + i) * hq + h) * HD + threadIdx.x] = Ls != 0.0f ? O / Ls : 0.0f;
    }
}

size_t tree_scratch_bytes(int n_seqs, int hq, int hkv, int max_seq_tokens, int max_ctx) { return 0; }

cudaError_t launch_paged_attn_tree(const float* q, const void* karena, const void* varena, int64_t n_arena_blocks,
                                   int n_layer, int layer, const int* bt, int mbs, const int* seq_starts,
                                   const int* ctx, const int64_t* mask, int words, int n_tok, int n_seqs,
                                   int max_seq_tokens, int hq, int hkv, int max_ctx, float scale, float* out,
                                   void* scratch, cudaStream_t st) {
    return launch_pdl(tree_simple_kernel, dim3((unsigned)max_seq_tokens, (unsigned)n_seqs, (unsigned)hq),
                      dim3(TREE_WARPS * 32), 0, st, q, (const __half*)karena, (const __half*)varena, n_arena_blocks,
                      n_layer, layer, bt, mbs, seq_starts, ctx, mask, words, n_tok, max_seq_tokens, hq, hkv,
                      scale * LOG2E, out);
}

}  // namespace dcg
