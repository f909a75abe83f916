// attn_tree.cu -- attention of a drafted token tree over DenseCore's paged fp16 KV cache.
//
// Beside the causal masks of the reference's attention selector (core/src/inference.cpp:1506-1573):
// drafted token i sees the whole history and, of the draft, the tokens whose bit is set in its mask
// row (its ancestors and itself).  Layout and checks as attn.cu.
//
// The (token, query head) pairs that share a kv head are the rows of one matrix: every K/V byte is
// read once for up to 128 of them.  An item is (sequence, kv head, tile of 128 rows), a unit one tile
// of 128 keys of an item; the units of the whole batch, in order, are cut into one range of equal cost
// per CTA (one CTA per SM), so ragged contexts load every SM alike.  Items that a range cuts leave
// their parts (unnormalised output, max, sum) in scratch; tree_combine_kernel joins them in CTA order.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <math.h>

#include "../../include/dcgpu.h"
#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace dcg {

constexpr int HD = 128;
constexpr int KVB = 16;
constexpr float LOG2E = 1.4426950408889634f;

__device__ int g_tree_error = 0;

cudaError_t tree_device_error(int* out, bool clear) {
    cudaError_t e = cudaMemcpyFromSymbol(out, g_tree_error, sizeof(int));
    if (e == cudaSuccess && clear && *out) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_tree_error, &zero, sizeof(int));
    }
    return e;
}

struct TreeArgs {
    const float* q;
    int64_t n_arena_blocks;
    int n_layer, layer;
    const int* bt;
    int mbs;
    const int *starts, *ctx;
    const int64_t* mask;
    int words, n_tok, n_seqs, max_tok, max_ctx, hq, hkv, nrep;
    float scale_log2;
    float* out;
    // scratch
    float *part_o, *part_ml;     // [2 G][rows][128], [2 G][rows][2]
    struct TreeCut* cuts;        // [G]
    struct TreeStart* begins;    // [G]
    int64_t* prefix;             // [2][n_seqs]: costs and units before each sequence
    int64_t* bounds;             // [G + 1]: first unit of each CTA
    int G;
    int part_rows;               // rows of the largest row tile
    int q_rows;                  // the same in eights (up to TW_STACK of them: sixteens): rows of a Q tile
    int row_tiles;               // of the largest sequence
    uint8_t* q_tiles;            // [n_seqs][row_tiles][hkv] x q_rows * 512 B: Q as halves, as shared memory wants it
    int8_t* q_exps;              // the same x q_rows: exponents of the rows' scales
};

// an item that CTA c begins and later CTAs go on with (rows = 0: none)
struct TreeCut {
    int rows, s0, row0, kvh;
    int parts;                   // CTAs that worked on it: c, c + 1, ...
};

// ---- the batch's units ----
struct TreeSeq {
    int s0, ns, L, tiles, row_tiles;
};
template <int ROWS, int KEYS>
__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs& a, int seq, bool report) {
    TreeSeq s;
    s.s0 = a.starts[seq];
    s.ns = a.starts[seq + 1] - s.s0;
    s.L = a.ctx[seq];
    const bool bad = s.s0 < 0 || s.ns < 0 || s.s0 > a.n_tok - s.ns || s.ns > a.max_tok || s.L < s.ns || s.L > a.max_ctx;
    if (bad) {
        if (report) atomicExch(&g_tree_error, DCG_DEVERR_INDEX);
        s.ns = s.L = 0;
    }
    s.tiles = s.ns ? (s.L + KEYS - 1) / KEYS : 0;
    s.row_tiles = (s.ns * a.nrep + ROWS - 1) / ROWS;
    return s;
}

// consecutive tiles of one item in a CTA's range
struct TreeSeg {
    int seq, kvh, rt, rows;      // rows of this row tile
    int tile0, tiles;            // of the item's
    TreeSeq s, next;             // next: of sequence seq + 1, its loads on the way meanwhile
    int left;                    // units of the range behind this segment
};
template <int ROWS, int KEYS>
__device__ __forceinline__ TreeSeq seq_or_none(const TreeArgs& a, int seq) {
    return seq < a.n_seqs ? tree_seq<ROWS, KEYS>(a, seq, false) : TreeSeq{0, 0, 0, 0, 0};
}
template <int ROWS>
__device__ __forceinline__ void seg_shape(const TreeArgs& a, TreeSeg& g) {
    g.rows = min(ROWS, g.s.ns * a.nrep - g.rt * ROWS);
    g.tiles = min(g.s.tiles - g.tile0, g.left);
    g.left -= g.tiles;
}
template <int ROWS, int KEYS>
__device__ __forceinline__ bool seg_next(const TreeArgs& a, TreeSeg& g) {
    if (g.left <= 0) return false;
    g.tile0 = 0;
    if (++g.rt == g.s.row_tiles) {
        g.rt = 0;
        if (++g.kvh == a.hkv) {
            g.kvh = 0;
            do {
                g.s = g.next;
                g.next = seq_or_none<ROWS, KEYS>(a, ++g.seq + 1);
            } while (!g.s.tiles);   // ends: units are left
        }
    }
    seg_shape<ROWS>(a, g);
    return true;
}

// where a CTA's range begins
struct TreeStart {
    int N;                       // its units
    int64_t u0;                  // its first unit
    TreeSeg g;
};

// Every CTA's range, by one CTA of THREADS.  An item costs its units and `extra` for its beginning, its
// masked last units and its output; the ranges cut the summed costs into equal parts, and a cut that
// falls into an item's extra cost goes to its first unit.  (A CTA inside an item has a unit at least, so
// an item's CTAs are consecutive.)
// Up to THREADS sequences the search runs in shared memory (a chain of global loads cost 3 us).
template <int ROWS, int KEYS, int THREADS>
__device__ void tree_plan_ranges(const TreeArgs& a, int extra) {
    __shared__ int64_t sums[2][THREADS / 32], s_cost[THREADS], s_units[THREADS], s_begin[THREADS];
    __shared__ TreeSeq s_seq[THREADS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool small = a.n_seqs <= THREADS;
    int64_t *cost = small ? s_cost : a.prefix, *units = small ? s_units : a.prefix + a.n_seqs;
    int64_t run = 0, run_u = 0;
    for (int i0 = 0; i0 < a.n_seqs; i0 += THREADS) {
        const int i = i0 + threadIdx.x;
        int64_t items = 0, u = 0;
        if (i < a.n_seqs) {
            const TreeSeq s = tree_seq<ROWS, KEYS>(a, i, true);
            items = s.tiles ? (int64_t)s.row_tiles * a.hkv : 0;
            u = s.tiles * items;
            if (small) s_seq[i] = s;
        }
        const int64_t c = u + extra * items;
        int64_t x = c, y = u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t p = __shfl_up_sync(0xffffffffu, x, o), q = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) {
                x += p;
                y += q;
            }
        }
        __syncthreads();
        if (lane == 31) {
            sums[0][warp] = x;
            sums[1][warp] = y;
        }
        __syncthreads();
        int64_t before = run, before_u = run_u;
#pragma unroll
        for (int w = 0; w < THREADS / 32; w++) {
            if (w < warp) {
                before += sums[0][w];
                before_u += sums[1][w];
            }
            run += sums[0][w];
            run_u += sums[1][w];
        }
        if (i < a.n_seqs) {
            cost[i] = before + x - c;
            units[i] = before_u + y - u;
        }
    }
    const int64_t V = run;
    const int G = (int)min((int64_t)a.G, V);      // no more ranges than cost: none is empty inside an item
    __syncthreads();
    auto seq_at = [&](int i) { return i >= a.n_seqs ? TreeSeq{0, 0, 0, 0, 0} : small ? s_seq[i] : tree_seq<ROWS, KEYS>(a, i, false); };
    // a range per thread: its first unit, and where that lies (a.G < THREADS)
    const int c = threadIdx.x;
    TreeStart b = {};
    b.u0 = run_u;
    if (c < G) {
        const int64_t v = sk_begin(c, V, G);
        int lo = 0, hi = a.n_seqs;                 // the last sequence that begins at or before v
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (cost[mid] <= v) lo = mid;
            else hi = mid;
        }
        b.g.seq = lo;
        b.g.s = seq_at(lo);
        const int off = (int)(v - cost[lo]), each = b.g.s.tiles + extra, item = off / each;
        b.g.tile0 = max(0, off - item * each - extra);
        b.g.kvh = item / b.g.s.row_tiles;
        b.g.rt = item - b.g.kvh * b.g.s.row_tiles;
        b.u0 = units[lo] + (int64_t)item * b.g.s.tiles + b.g.tile0;
    }
    s_begin[c] = b.u0;
    __syncthreads();
    if (c > a.G) return;
    a.bounds[c] = b.u0;
    if (c == a.G) return;
    b.N = (int)(s_begin[c + 1] - b.u0);
    b.g.left = b.N;
    if (b.N) {
        b.g.next = seq_at(b.g.seq + 1);
        seg_shape<ROWS>(a, b.g);
    }
    a.begins[c] = b;
    a.cuts[c].rows = 0;
}

// mask bits of keys g0 .. g0 + 31 (as positions) for the drafted token of mask row `m`, whose first word
// is m0: history, then draft
__device__ __forceinline__ uint32_t tree_bits(const TreeArgs& a, const TreeSeq& s, const uint64_t* m, uint64_t m0, int g0) {
    const int hist = s.L - s.ns, t0 = g0 - hist;
    if (t0 <= -32) return 0xFFFFFFFFu;
    if (g0 >= s.L) return 0u;
    uint32_t v;
    if (t0 < 0) {
        v = (uint32_t)(m0 << -t0) | ((1u << -t0) - 1);
    } else {
        const int w = t0 >> 6, b = t0 & 63;
        v = (uint32_t)((w ? m[w] : m0) >> b);
        if (b > 32 && w + 1 < a.words) v |= (uint32_t)(m[w + 1] << (64 - b));
    }
    const int n = s.L - g0;
    return n >= 32 ? v : v & ((1u << n) - 1);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_h2(float x0, float x1) {
    const __half2 h = __floats2half2_rn(x0, x1);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// x = hi + lo as fp16 halves (to 2^-21 of x): hi is x cut to 11 bits, so the rest is exact
__device__ __forceinline__ void cut_h2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const float h0 = __uint_as_float(__float_as_uint(x0) & 0xFFFFE000u), h1 = __uint_as_float(__float_as_uint(x1) & 0xFFFFE000u);
    hi = pack_h2(h0, h1);
    lo = pack_h2(x0 - h0, x1 - h1);
}

// ------------------------------------------------------------------------------------------
// tree_wide_kernel<STACKED>: tcgen05, one row tile x 128 keys per unit.
//   S = Q K^T: Q as two fp16 halves (hi + lo) in shared memory, each row scaled by a power of two so
//     that its largest value lies in [1, 2); K as it is in the cache.
//   p = 2^(c s - m + 8), c = scale log2(e) / row scale, m the tile's own row max; cut into halves that
//     overwrite S in tensor memory.
//   O = P V of this tile alone: A from tensor memory, V as it is in the cache (MN-major).
//   The tiles' O, m and sum of p are joined in registers, in fp32 rounded to nearest.
// Up to 128 rows an item: both halves into one accumulator, 16 + 16 MMAs of M128 N128 K16 a unit; k-step
// j's 8 + 8 columns of P lie where its 16 scores were.  STACKED, up to 64 rows: a row's halves are two rows
// of the MMA (64-row MMAs take as long as 128-row ones), 8 + 8 MMAs a unit, and the softmax reads
// fragments of 16 lanes, two halves added, 4 threads for 2 rows (98 -> 87 us for one sequence of 100,003
// tokens and 52 rows against 64-row MMAs).
// The tensor core cuts its sums off rather than rounding them, a bias of up to 2^-24 for each MMA that
// adds to a large accumulator: hence the lo halves first, and no accumulator that lives for longer
// than a tile (one that lived for a segment was 2-4 x 10^-6 off, this is 4-8 x 10^-7).
// Two S / P and two O buffers, used in turn.  Warps: 0 and 3 TMA producers of K (and each segment's Q,
// up to 64 rows into a second buffer) and V (one ring of 5 x 32 KB, in the order the MMAs take them;
// pages beyond the sequence load as zeros), 1 and 2 MMA issue for every other tile, 4-7 and 8-11 its
// softmax, 12-15 the running output (128 registers of it per thread, thread = row).  tree_q_kernel has laid Q out
// before: converting it here cost 20,000 cycles at every change of the item.
// What bounds it: a unit's chain S (700 cycles stacked, 1,470 not), softmax (2,500), O (650 / 1,250) in two
// streams, 2,400 cycles a stacked unit while items are long: 1.2 us at the full clock, where an SM's share of HBM is
// the limit (64 KB, 1.5 us), and 1.6 us at the 1.5 GHz of long runs, where the chain is; at an item's end
// 4,000 cycles more for masks, cleaning and the change.  Times with tree_q_kernel and
// tree_combine_kernel: 1 x 13 tokens, 100,003 of context 83 us (410 MB, 4.9 TB/s); 32 x 16, up to 2,048
// 49 us (163 MB); 16 x 64, 64 heads, up to 4,096 151 us (118 GFLOP with both halves, 780 TFLOP/s); sustained, at
// the power limit's clock, 100, 52 and 181 us.
// ------------------------------------------------------------------------------------------
constexpr int TW_ROWS = 128;
constexpr int TW_KEYS = 128;
constexpr int TW_STACK = 64;                      // up to so many rows an item: both halves in one accumulator
constexpr int TW_RING = 5;
constexpr int TW_BUF = TW_KEYS * HD * 2;          // 32 KB: [half of 64 dims][128 keys][128 B]
constexpr int TW_HALF = TW_BUF / 2;
constexpr int TW_THREADS = 512;
constexpr int TW_OFF_RING = 2 * TW_BUF;           // Q hi, Q lo first
constexpr int TW_OFF_CTRL = TW_OFF_RING + TW_RING * TW_BUF;
constexpr int TW_CTRL = 2560;
constexpr int TW_SMEM = TW_OFF_CTRL + TW_CTRL;    // of 227 KB
constexpr int TW_EXTRA = 4, TW_EXTRA_STACKED = 2; // an item's fixed cost in units (5.7 us against 1.4 us a unit; 2.4 and 1.1)
constexpr float TW_SHIFT = 8.0f;                  // p is at most 2^8: the small ones stay above fp16's least
// registers per thread of the four warpgroups (control, 2 x softmax, output): 512 of a launch's 4 x 128,
// as few spills as any split has
constexpr int tw_regs_ctrl(bool stacked) { return stacked ? 56 : 80; }
constexpr int TW_REGS_SOFT = 128;
constexpr int tw_regs_out(bool stacked) { return 512 - 2 * TW_REGS_SOFT - tw_regs_ctrl(stacked); }

struct TwCtrl {
    uint64_t full[TW_RING], empty[TW_RING], s_full[2], p_full[2], o_full[2], o_free[2], x_free[2], cleaned[2];
    uint64_t q_full[2], q_empty[2][2], mma_end[2];   // q_empty: by MMA warp and buffer
    uint32_t tmem;
    uint32_t bad[2][3][4];                        // per buffer, special tiles in turn: keys whose V is not finite
    float2 x[2][TW_ROWS];                         // a tile's row max and sum of p
};
static_assert(sizeof(TwCtrl) <= TW_CTRL, "control block");

__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, bool b_mn) {
    // D f32 (bits 4-5 = 1), A and B f16 (0), B MN-major (bit 16), N >> 3 at 17-22, M >> 4 at 24-28
    return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// whether phase `parity` of `bar` is over, without waiting
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return __all_sync(0xffffffffu, done != 0);
}
// one thread of the warp, the same each time
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
}
template <bool ACC>
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(ad), "l"(bd), "r"(idesc), "n"(ACC ? 1 : 0) : "memory");
}
template <bool ACC>
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t at, uint64_t bd, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(at), "l"(bd), "r"(idesc), "n"(ACC ? 1 : 0) : "memory");
}
// MN-major operand, 128-byte swizzle: rows of 64 MN-elements, 8-row (K) atoms 1 KB apart, the next 64
// MN-elements TW_HALF further
__device__ __forceinline__ uint64_t umma_desc_mn128(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(TW_HALF >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
          "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
          "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
          "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}

// 16 lanes (16 into `taddr`'s 32, or from them on) x 32 columns as fragments: thread t has of each 8 columns b
// row t / 4, columns 2 (t % 4) + {0, 1} in v[4 b], v[4 b + 1] and row t / 4 + 8 in the next two
__device__ __forceinline__ void tmem_ld_frag(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_frag32(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                 "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
// and 16 lanes x 16 columns: of each 4 columns b row t / 4, column t % 4 in v[2 b] and row t / 4 + 8 in v[2 b + 1]
__device__ __forceinline__ void tmem_st_frag(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

__device__ __forceinline__ void prefetch_tensormap(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)map) : "memory");
}
// ring position of the K and V tile of the range's n-th unit of N: K0 K1 V0 K2 V1 ... K(N-1) V(N-2) V(N-1)
__device__ __forceinline__ uint32_t tw_k(int n) { return n ? 2 * n - 1 : 0; }
__device__ __forceinline__ uint32_t tw_v(int n, int N) { return n == N - 1 ? 2 * N - 1 : 2 * n + 2; }

// two fp32 operations at a time
__device__ __forceinline__ uint64_t pack2(float x0, float x1) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x0), "f"(x1));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t r, float& x0, float& x1) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x0), "=f"(x1) : "l"(r)); }
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}

// Q as fp16 halves in the tiles that tree_wide_kernel copies: [hi, lo][half of 64 dims][q_rows][128 B], or
// stacked [half of 64 dims][16 rows hi, the same lo, the next 16 hi, ...][128 B];
// 128-byte swizzle, each row scaled by a power of two (its sign the scale's).  CTA (TQ_ROWS of a
// sequence's rows, which lie one behind the other; sequence), 8 lanes a row.  One CTA more plans the ranges.
constexpr int TQ_WARPS = 8, TQ_ROWS = 64;
__global__ void __launch_bounds__(TQ_WARPS * 32) tree_q_kernel(const TreeArgs a) {
    __shared__ __align__(128) float rows[TQ_ROWS * HD];
    __shared__ uint64_t bar;
    pdl_wait();
    pdl_trigger();
    if (blockIdx.y == 0) {                        // first in the launch order
        if (blockIdx.x == 0) tree_plan_ranges<TW_ROWS, TW_KEYS, TQ_WARPS * 32>(a, a.q_rows <= TW_STACK ? TW_EXTRA_STACKED : TW_EXTRA);
        return;
    }
    const int seq = blockIdx.y - 1;
    const TreeSeq s = tree_seq<TW_ROWS, TW_KEYS>(a, seq, false);
    const int x0 = blockIdx.x * TQ_ROWS, n = min(TQ_ROWS, s.ns * a.hq - x0), lane = threadIdx.x & 31;
    const int to = s.row_tiles ? (s.row_tiles - 1) * TW_ROWS + a.q_rows : 0;   // rows that tree_wide_kernel reads
    if (x0 / a.hq * a.nrep >= to) return;
    if (threadIdx.x == 0 && n > 0) {
        mbar_init(&bar, 1);
        fence_mbar_init();
        mbar_arrive_expect_tx(&bar, (uint32_t)n * HD * 4);
        bulk_g2s(rows, a.q + ((int64_t)s.s0 * a.hq + x0) * HD, (uint32_t)n * HD * 4, &bar);
    }
    __syncthreads();
    const bool stacked = a.q_rows <= TW_STACK;
    const int dims_half = a.q_rows * (stacked ? 256 : 128), to_lo = stacked ? 16 * 128 : a.q_rows * 256;
    if (n > 0 && !mbar_wait(&bar, 0, &g_tree_error)) return;
#pragma unroll 1
    for (int i0 = (threadIdx.x >> 5) * 4; i0 < TQ_ROWS; i0 += TQ_WARPS * 4) {
        const int i = i0 + (lane >> 3), sub = lane & 7;
        const int t = (x0 + i) / a.hq, h = x0 + i - t * a.hq;
        const int kvh = h / a.nrep, R = t * a.nrep + h - kvh * a.nrep, rt = R / TW_ROWS, r = R - rt * TW_ROWS;
        const int64_t tile = ((int64_t)seq * a.row_tiles + rt) * a.hkv + kvh;
        float x[2][8], m = 0.0f;                  // dims 8 sub .. +7 of both halves; zeros behind the last query
#pragma unroll
        for (int d = 0; d < 2; d++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const float4 y = i < n ? *(const float4*)(rows + i * HD + 64 * d + 8 * sub + 4 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
                x[d][4 * c] = y.x;
                x[d][4 * c + 1] = y.y;
                x[d][4 * c + 2] = y.z;
                x[d][4 * c + 3] = y.w;
                m = fmaxf(fmaxf(m, fmaxf(fabsf(y.x), fabsf(y.y))), fmaxf(fabsf(y.z), fabsf(y.w)));
            }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (R >= to) continue;
        // exponent of the row's largest value (0 rows and subnormal ones: the least)
        int e = (int)(__float_as_uint(m) >> 23) - 127;
        e = e < -100 ? -100 : e > 120 ? 120 : e;
        const float f = copysignf(__uint_as_float((uint32_t)(127 - e) << 23), a.scale_log2);   // 2^-e
        const int at = stacked ? 2 * r - (r & 15) : r;
        uint8_t* dst = a.q_tiles + tile * a.q_rows * 512 + at * 128 + ((sub ^ (r & 7)) << 4);
#pragma unroll
        for (int d = 0; d < 2; d++) {
            uint4 hi, lo;
            cut_h2(x[d][0] * f, x[d][1] * f, hi.x, lo.x);
            cut_h2(x[d][2] * f, x[d][3] * f, hi.y, lo.y);
            cut_h2(x[d][4] * f, x[d][5] * f, hi.z, lo.z);
            cut_h2(x[d][6] * f, x[d][7] * f, hi.w, lo.w);
            *(uint4*)(dst + d * dims_half) = hi;
            *(uint4*)(dst + d * dims_half + to_lo) = lo;
        }
        if (sub == 0) a.q_exps[tile * a.q_rows + r] = (int8_t)e;
    }
}

// STACKED: every item has at most 64 rows.  Row r = 16 q + i has its hi half in lane 32 q + i of the MMAs'
// 128 and its lo half in lane 32 q + 16 + i, so 8 + 8 MMAs make a unit; S is the two lanes' sum, and so is O.
template <bool STACKED>
__global__ void __launch_bounds__(TW_THREADS, 1) tree_wide_kernel(
    const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const TreeArgs a) {
    extern __shared__ __align__(1024) uint8_t smem[];   // no static shared memory: starts on a KB
    uint8_t* ring = smem + TW_OFF_RING;
    TwCtrl& C = *(TwCtrl*)(smem + TW_OFF_CTRL);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (smem_u32(smem) & 1023) {                  // the swizzled tiles would not match their descriptors
        if (threadIdx.x == 0) atomicExch(&g_tree_error, DCG_DEVERR_TIMEOUT);
        return;
    }

    if (threadIdx.x == 0) {
        for (int s = 0; s < TW_RING; s++) {
            mbar_init(&C.full[s], 1);
            mbar_init(&C.empty[s], 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&C.s_full[b], 1);
            mbar_init(&C.p_full[b], 4);
            mbar_init(&C.o_full[b], 1);
            mbar_init(&C.o_free[b], 4);
            mbar_init(&C.x_free[b], 4);
            mbar_init(&C.cleaned[b], 4);
            mbar_init(&C.q_full[b], 1);
            mbar_init(&C.q_empty[0][b], 1);
            mbar_init(&C.q_empty[1][b], 1);
            mbar_init(&C.mma_end[b], 1);
        }
        fence_mbar_init();
    }
    if (threadIdx.x < 24) (&C.bad[0][0][0])[threadIdx.x] = 0;
    if (STACKED) {                                // rows without a query stay zeros: the tensor core's power is the limit
        for (int i = threadIdx.x; i < 2 * TW_BUF / 16; i += TW_THREADS) ((uint4*)smem)[i] = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&C.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (threadIdx.x == 0 || threadIdx.x == 96) prefetch_tensormap(threadIdx.x ? &vmap : &kmap);
    pdl_wait();
    pdl_trigger();                                // tree_combine_kernel's CTAs wait where this one's have ended
    const TreeStart& start = a.begins[blockIdx.x];
    const int N = start.N;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = C.tmem;
    bool ok = true;

    constexpr int q_bufs = STACKED ? 2 : 1;       // as many as there is room for
    const int q_bytes = a.q_rows * 512, q_buf = STACKED ? TW_BUF : q_bytes;
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(tw_regs_ctrl(STACKED)));
        if (N == 0) {
        } else if (warp == 0 || warp == 3) {
            // ---------------- Q and K tiles (warp 0), V tiles (warp 3) ----------------
            // 16 boxes of 2 KB a tile, one for each of 16 lanes: a warp issues one in about 80 cycles
            const bool is_v = warp == 3;
            const CUtensorMap* map = is_v ? &vmap : &kmap;
            TreeSeg g = start.g;
            const int page = lane >> 1, half = lane & 1;
            const int beyond = (int)(a.n_arena_blocks * a.n_layer * KVB);   // out of the arena: zeros
            // block id of this lane's page in a tile, INT32_MIN behind the sequence's end (no read)
            auto block = [&](const TreeSeg& s, int tile) {
                const int p = (s.tile0 + tile) * (TW_KEYS / KVB) + page;
                return lane < 16 && p * KVB < s.s.L ? a.bt[(int64_t)s.seq * a.mbs + p] : INT32_MIN;
            };
            int t = 0, b = block(g, 0), kvh = g.kvh, n = 0, seg = 0;
            bool begins = true;
            for (; n < N; n++) {
                const uint32_t l = is_v ? tw_v(n, N) : tw_k(n), slot = l % TW_RING;
                const bool in = b >= 0 && b < a.n_arena_blocks;
                if (!in && b != INT32_MIN) atomicExch(&g_tree_error, DCG_DEVERR_INDEX);
                const int row = in ? (b * a.n_layer + a.layer) * KVB : beyond, head = kvh;
                if (begins && !is_v) {             // the segment's Q, ahead of its first K
                    const int qb = seg % q_bufs;
                    const int64_t q_tile = ((int64_t)g.seq * a.row_tiles + g.rt) * a.hkv + g.kvh;
                    ok = __all_sync(0xffffffffu, seg < q_bufs || mbar_wait(&C.q_empty[lane & 1][qb], (uint32_t)((seg / q_bufs - 1) & 1), &g_tree_error));
                    if (!ok) break;
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&C.q_full[qb], (uint32_t)q_bytes);
                        for (int d = 0; d < (STACKED ? 2 : 1); d++)
                            bulk_g2s(smem + qb * q_buf + d * TW_HALF, a.q_tiles + q_tile * q_bytes + d * (q_bytes / 2),
                                     (uint32_t)(STACKED ? q_bytes / 2 : q_bytes), &C.q_full[qb]);
                    }
                    seg++;
                }
                begins = false;
                if (++t == g.tiles) {
                    t = 0;
                    begins = true;
                    if (n + 1 < N) seg_next<TW_ROWS, TW_KEYS>(a, g);
                }
                if (n + 1 < N) {                   // on its way while the ring is waited for
                    b = block(g, t);
                    kvh = g.kvh;
                }
                ok = __all_sync(0xffffffffu, l < TW_RING || mbar_wait(&C.empty[slot], (l / TW_RING - 1) & 1, &g_tree_error));
                if (!ok) break;
                if (lane == 0) mbar_arrive_expect_tx(&C.full[slot], TW_BUF);
                __syncwarp();
                if (lane < 16) tma_load_4d(ring + (size_t)slot * TW_BUF + half * TW_HALF + page * 2048, map, 0, row, half, head, &C.full[slot]);
            }
            if (!ok) {                             // given up: the copies in flight land before the CTA ends
                if (!is_v)
                    for (int i = max(0, seg - q_bufs); i < seg; i++) mbar_wait(&C.q_full[i % q_bufs], (uint32_t)((i / q_bufs) & 1), &g_tree_error, 1u << 16);
                for (int i = max(0, n - TW_RING); i < n; i++) {
                    const uint32_t l = is_v ? tw_v(i, N) : tw_k(i);
                    mbar_wait(&C.full[l % TW_RING], (l / TW_RING) & 1, &g_tree_error, 1u << 16);
                }
            }
        } else {
            // ---------------- MMA issue: warp 1 the even units, warp 2 the odd ones ----------------
            // Each in step, one elected thread issuing.  A warp's polls, and its waits for the tensor core to
            // take its last operands, leave the core with the other's work.
            constexpr uint32_t id_s = idesc_f16(TW_ROWS, TW_KEYS, false), id_o = idesc_f16(TW_ROWS, HD, true);
            const uint32_t qs = smem_u32(smem), rg = qs + TW_OFF_RING, q_half = STACKED ? TW_HALF : a.q_rows * 128;
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            const bool leader = elect_one();
            const int b = warp - 1;
            const uint32_t S = tm + b * 128, O = tm + 256 + b * 128;   // P takes S's place
            TreeSeg g = start.g;
            int seg = 0, end = g.tiles;            // the segment's end among the range's units
            bool begins = true;                    // its Q not waited for yet
            uint64_t* q_empty = C.q_empty[b];
            // S of unit n
            auto issue_s = [&](int n, bool have_k) {
                while (n >= end) {                 // (a segment that has no unit of this warp: given back at once)
                    if (begins && leader) tc_commit(&q_empty[seg % q_bufs]);
                    seg_next<TW_ROWS, TW_KEYS>(a, g);
                    seg++;
                    end += g.tiles;
                    begins = true;
                }
                const int qb = seg % q_bufs;
                const uint32_t l = tw_k(n), slot = l % TW_RING;
                uint64_t* bar = lane == 0 ? &C.q_full[qb] : &C.full[slot];
                const uint32_t parity = lane == 0 ? (uint32_t)((seg / q_bufs) & 1) : (l / TW_RING) & 1;
                if (begins || !have_k) {
                    ok = __all_sync(0xffffffffu, (lane == 0 && !begins) || mbar_wait(bar, parity, &g_tree_error));
                    if (!ok) return;
                    begins = false;
                    tc_fence_after();
                }
                if (leader) {
                    const uint32_t q = qs + qb * q_buf;
                    const uint64_t kd = umma_desc_sw128(rg + slot * TW_BUF);
#pragma unroll
                    for (int h = STACKED ? 0 : 1; h >= 0; h--) {   // the lo half first
#pragma unroll
                        for (int d = 0; d < 2; d++) {
                            const uint64_t qd = umma_desc_sw128(q + (2 * h + d) * q_half);
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                if (h == !STACKED && !d && j == 0) mma_f16_ss<false>(S, qd + 2 * j, kd + d * (TW_HALF >> 4) + 2 * j, id_s);
                                else mma_f16_ss<true>(S, qd + 2 * j, kd + d * (TW_HALF >> 4) + 2 * j, id_s);
                            }
                        }
                    }
                    tc_commit(&C.s_full[b]);
                    tc_commit(&C.empty[slot]);
                    if (n + 2 >= end) tc_commit(&q_empty[qb]);
                }
                __syncwarp();
            };
            // No S is issued before the one ahead of it has ended (below, by lane 2's wait).  So every Q up to then, and
            // every K, has landed, also of segments and units that are the other warp's: a barrier that has ended no
            // phase passes a wait for its second one, which has the same parity.
            if (b && b < N) ok = __all_sync(0xffffffffu, mbar_wait(&C.s_full[0], 0, &g_tree_error));
            if (b < N && ok) issue_s(b, false);
            for (int n = b; n < N && ok; n += 2) {  // O of unit n, then S of unit n + 2 into the same buffer
                const uint32_t k = (uint32_t)n >> 1, l = tw_v(n, N), slot = l % TW_RING;
                // one poll for all: lane 0 V, 1 O's buffer, 2 S of the next unit, others P.  (The third keeps the
                // two streams apart, and the tiles' order: a slot of the ring holds K and V in turn, and a producer
                // that came a fill too early would not see it by the parity.)
                uint64_t* bar = &C.p_full[b];
                uint32_t parity = k & 1;
                bool wait = true;
                if (lane == 0) {
                    bar = &C.full[slot];
                    parity = (l / TW_RING) & 1;
                } else if (lane == 1) {
                    bar = &C.o_free[b];
                    parity = (k - 1) & 1;
                    wait = k > 0;
                } else if (lane == 2) {
                    bar = &C.s_full[b ^ 1];
                    parity = ((uint32_t)(n + 1) >> 1) & 1;
                    wait = n + 1 < N;
                }
                ok = __all_sync(0xffffffffu, !wait || mbar_wait(bar, parity, &g_tree_error));
                if (!ok) break;
                const uint32_t lk = tw_k(n + 2);   // S of unit n + 2 follows at once if its K is there
                const bool have_k = n + 2 < N && mbar_test(&C.full[lk % TW_RING], (lk / TW_RING) & 1);
                tc_fence_after();
                if (leader) {
                    const uint64_t vd = umma_desc_mn128(rg + slot * TW_BUF);
#pragma unroll
                    for (int h = STACKED ? 0 : 1; h >= 0; h--)   // 16 keys = 2048 bytes per k-step
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const uint32_t P = S + (STACKED ? 8 : 16) * j + 8 * h;
                            if (h == !STACKED && j == 0) mma_f16_ts<false>(O, P, vd + j * (2048 >> 4), id_o);
                            else mma_f16_ts<true>(O, P, vd + j * (2048 >> 4), id_o);
                        }
                    tc_commit(&C.o_full[b]);
                    tc_commit(&C.empty[slot]);
                }
                __syncwarp();
                if (n + 2 < N) issue_s(n + 2, have_k);
            }
            if (leader) tc_commit(&C.mma_end[b]);
            __syncwarp();
            mbar_wait(&C.mma_end[b], 0, &g_tree_error);
        }
    } else if (warp < 12) {
        // ---------------- softmax of every other tile (thread = row; stacked: 4 threads for 2 rows) ----------------
        const int wg = (warp - 4) >> 2, quad = warp & 3, tid = quad * 32 + lane;
        const int r = STACKED ? quad * 16 + (lane & 15) : tid;
        const int r0 = quad * 16 + (lane >> 2), r1 = r0 + 8;   // stacked: the rows of this thread's fragments
        const uint32_t S = tmem + ((uint32_t)(quad * 32) << 16) + wg * 128;
        uint32_t cleans = 0;
        int n = 0;
        if (N) {
            TreeSeg g = start.g;
            do {
                const bool valid = r < g.rows, live = quad * (STACKED ? 16 : 32) < g.rows;
                const int hist = g.s.L - g.s.ns;
                const uint64_t* mask = (const uint64_t*)a.mask + (int64_t)(g.s.s0 + (valid ? (g.rt * TW_ROWS + r) / a.nrep : 0)) * a.words;
                const uint64_t mask0 = *mask;
                // c > 0 (the scale's sign is in Q), and not 0: c x -inf has to stay -inf
                const int64_t tile = ((int64_t)g.seq * a.row_tiles + g.rt) * a.hkv + g.kvh;
                auto scale = [&](int row) {
                    const int qexp = row < g.rows ? a.q_exps[tile * a.q_rows + row] : 0;
                    return fmaxf(fabsf(a.scale_log2) * __uint_as_float((uint32_t)(127 + qexp) << 23), 1e-37f);
                };
                const float c = scale(STACKED ? r0 : r), c1 = STACKED ? scale(r1) : c;
                for (int t = 0; t < g.tiles && ok; t++, n++) {
                    if ((int)(n & 1) != wg) continue;
                    const uint32_t k = (uint32_t)(n >> 1);
                    ok = __all_sync(0xffffffffu, mbar_wait(&C.s_full[wg], k & 1, &g_tree_error));
                    if (!ok) break;
                    tc_fence_after();
                    const int kb = (g.tile0 + t) * TW_KEYS;
                    const bool special = kb + TW_KEYS > hist;
                    uint32_t vis[2];                       // stacked: lane i and i + 16 the first and last 64 keys of row i
                    if (special && live) {                 // -inf for the keys that a row does not see
                        auto bits = [&](int w) { return valid ? tree_bits(a, g.s, mask, mask0, kb + 32 * w) : 0u; };
                        if (STACKED) {
#pragma unroll 1
                            for (int w = 0; w < 2; w++) {
                                const uint32_t v = bits(2 * (lane >> 4) + w);
                                if (w) vis[1] = v;
                                else vis[0] = v;
                            }
                        }
#pragma unroll 1
                        for (int w = 0; w < 4; w++) {
                            if (STACKED) {
                                uint32_t hi[16], lo[16];
                                tmem_ld_frag(S + 32 * w, hi);
                                tmem_ld_frag(S + (16u << 16) + 32 * w, lo);
                                const int from = (lane >> 2) + 16 * (w >> 1);
                                const uint32_t v = w & 1 ? vis[1] : vis[0];
                                const uint32_t v0 = __shfl_sync(0xffffffffu, v, from) >> (2 * (lane & 3));
                                const uint32_t v1 = __shfl_sync(0xffffffffu, v, from + 8) >> (2 * (lane & 3));
                                tmem_wait_ld();
#pragma unroll
                                for (int i = 0; i < 16; i++)
                                    if (!(((i & 2 ? v1 : v0) >> (8 * (i >> 2) + (i & 1))) & 1)) {
                                        hi[i] = 0xFF800000u;
                                        lo[i] = 0u;
                                    }
                                tmem_st_frag32(S + 32 * w, hi);
                                tmem_st_frag32(S + (16u << 16) + 32 * w, lo);
                            } else {
                                const uint32_t v = bits(w);
                                uint32_t s[32];
                                tmem_ld32(S + 32 * w, s);
                                tmem_wait_ld();
#pragma unroll
                                for (int i = 0; i < 32; i++) s[i] = (v >> i) & 1 ? s[i] : 0xFF800000u;
                                tmem_st32(S + 32 * w, s);
                            }
                        }
                        tmem_wait_st();
                    }
                    float m = -INFINITY, sum = 0.0f, m1 = -INFINITY, sum1 = 0.0f;
                    if (STACKED && live) {
                        // rolled loops: the code of all the warps has to stay in the instruction cache
                        uint32_t hi[16], lo[16];           // the next 32 scores, loaded while x is worked on
                        float x[16];
                        tmem_ld_frag(S, hi);
                        tmem_ld_frag(S + (16u << 16), lo);
                        auto scores = [&](int w, bool more) {
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; i += 2)
                                unpack2(add2(pack2(__uint_as_float(hi[i]), __uint_as_float(hi[i + 1])),
                                             pack2(__uint_as_float(lo[i]), __uint_as_float(lo[i + 1]))), x[i], x[i + 1]);
                            if (more) {
                                tmem_ld_frag(S + 32 * ((w + 1) & 3), hi);
                                tmem_ld_frag(S + (16u << 16) + 32 * ((w + 1) & 3), lo);
                            }
                        };
                        float y[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
                        for (int w = 0; w < 4; w++) {
                            scores(w, true);
#pragma unroll
                            for (int i = 0; i < 16; i++) y[i & 3] = fmaxf(y[i & 3], x[i]);
                        }
                        y[0] = fmaxf(y[0], y[1]);
                        y[2] = fmaxf(y[2], y[3]);
#pragma unroll
                        for (int o = 1; o < 4; o <<= 1) {
                            y[0] = fmaxf(y[0], __shfl_xor_sync(0xffffffffu, y[0], o));
                            y[2] = fmaxf(y[2], __shfl_xor_sync(0xffffffffu, y[2], o));
                        }
                        m = y[0] * c;
                        m1 = y[2] * c1;
                        // (rows without a query: p = 0)
                        const float sh0 = r0 < g.rows ? TW_SHIFT - (m == -INFINITY ? 0.0f : m) : -INFINITY;
                        const float sh1 = r1 < g.rows ? TW_SHIFT - (m1 == -INFINITY ? 0.0f : m1) : -INFINITY;
                        const uint64_t k2[2] = {pack2(c, c), pack2(c1, c1)}, h2[2] = {pack2(sh0, sh0), pack2(sh1, sh1)};
                        uint64_t sum2[2] = {0, 0};
#pragma unroll 1
                        for (int w = 0; w < 4; w++) {      // P's columns lie behind the scores still to be read
                            scores(w, w < 3);
                            uint32_t ph[8], pl[8];
#pragma unroll
                            for (int i = 0; i < 8; i++) {
                                float p0, p1;
                                unpack2(fma2(pack2(x[2 * i], x[2 * i + 1]), k2[i & 1], h2[i & 1]), p0, p1);
                                p0 = ex2(p0);
                                p1 = ex2(p1);
                                sum2[i & 1] = add2(sum2[i & 1], pack2(p0, p1));
                                cut_h2(p0, p1, ph[i], pl[i]);
                            }
                            tmem_st_frag(S + 16 * w, ph);
                            tmem_st_frag(S + (16u << 16) + 16 * w, pl);
                        }
                        unpack2(sum2[0], y[0], y[1]);
                        unpack2(sum2[1], y[2], y[3]);
                        sum = y[0] + y[1];
                        sum1 = y[2] + y[3];
#pragma unroll
                        for (int o = 1; o < 4; o <<= 1) {
                            sum += __shfl_xor_sync(0xffffffffu, sum, o);
                            sum1 += __shfl_xor_sync(0xffffffffu, sum1, o);
                        }
                    } else if (live) {
                        // rolled loops: the two warpgroups' code has to stay in the instruction cache
                        float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
                        for (int w = 0; w < 4; w += 2) {
                            uint32_t s[2][32];
                            tmem_ld32(S + 32 * w, s[0]);
                            tmem_ld32(S + 32 * w + 32, s[1]);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i += 4)
#pragma unroll
                                for (int e = 0; e < 4; e++)
                                    x[e] = fmaxf(x[e], fmaxf(__uint_as_float(s[0][i + e]), __uint_as_float(s[1][i + e])));
                        }
                        const float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                        m = mx * c;
                        const float shift = TW_SHIFT - (m == -INFINITY ? 0.0f : m);
                        const uint64_t c2 = pack2(c, c), h2 = pack2(shift, shift);
                        uint64_t sum2 = 0;
                        // 32 scores -> p as halves, in their place
                        auto halves = [&](uint32_t (&s)[32]) {
#pragma unroll
                            for (int j = 0; j < 2; j++) {
                                uint32_t hi[8], lo[8];
#pragma unroll
                                for (int i = 0; i < 8; i++) {
                                    const int e = 16 * j + 2 * i;
                                    float p0, p1;
                                    unpack2(fma2(pack2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), c2, h2), p0, p1);
                                    p0 = ex2(p0);
                                    p1 = ex2(p1);
                                    sum2 = add2(sum2, pack2(p0, p1));
                                    cut_h2(p0, p1, hi[i], lo[i]);
                                }
#pragma unroll
                                for (int i = 0; i < 8; i++) {
                                    s[16 * j + i] = hi[i];
                                    s[16 * j + 8 + i] = lo[i];
                                }
                            }
                        };
                        uint32_t s0[32], s1[32];           // one is loaded while the other is worked on
                        tmem_ld32(S, s0);
#pragma unroll 1
                        for (int w = 0; w < 4; w += 2) {
                            tmem_wait_ld();
                            tmem_ld32(S + 32 * w + 32, s1);
                            halves(s0);
                            tmem_st32(S + 32 * w, s0);
                            tmem_wait_ld();
                            if (w == 0) tmem_ld32(S + 64, s0);
                            halves(s1);
                            tmem_st32(S + 32 * w + 32, s1);
                        }
                        float odd;
                        unpack2(sum2, sum, odd);
                        sum += odd;
                    }
                    if (special) {                         // behind the softmax, which V need not wait for
                        // V of slots past the context may be anything, and that of a drafted token that
                        // this row does not see may be NaN: 0 x NaN is NaN, so such V become zeros
                        const uint32_t lv = tw_v(n, N);
                        ok = __all_sync(0xffffffffu, mbar_wait(&C.full[lv % TW_RING], (lv / TW_RING) & 1, &g_tree_error));
                        if (!ok) break;
                        // (pages past the sequence's last came as zeros).  A chunk of 16 bytes per lane, two keys
                        // at a time, the warps in turn.
                        uint32_t* bad = C.bad[wg][cleans % 3];
                        if (tid < 4) C.bad[wg][(cleans + 1) % 3][tid] = 0;   // the last but one's: all have read it
                        uint8_t* v = ring + (lv % TW_RING) * TW_BUF + ((lane >> 3) & 1) * TW_HALF + (lane & 7) * 16;
                        const int end = min((g.s.L + KVB - 1) / KVB * KVB - kb, TW_KEYS);
#pragma unroll 1
                        for (int i = max(hist - kb, 0) / 2 + quad; 2 * i < end; i += 4) {
                            const int key = 2 * i + (lane >> 4);
                            uint4* chunk = (uint4*)(v + key * 128);
                            bool odd = false;
                            if (kb + key >= hist && kb + key < g.s.L) {
                                const uint4 w = *chunk;
                                const uint32_t y[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                                for (int e = 0; e < 4; e++)
                                    odd |= (y[e] & 0x7C00u) == 0x7C00u || (y[e] & 0x7C000000u) == 0x7C000000u;
                            }
                            const bool any = (__ballot_sync(0xffffffffu, odd) >> (lane & 16)) & 0xFFFFu;
                            if (any || kb + key >= g.s.L) *chunk = make_uint4(0, 0, 0, 0);
                            if (any && (lane & 15) == 0) atomicOr(&bad[key >> 5], 1u << (key & 31));
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&C.cleaned[wg]);
                        ok = __all_sync(0xffffffffu, mbar_wait(&C.cleaned[wg], cleans++ & 1, &g_tree_error));
                        if (!ok) break;
                        if (live) {                        // a row that sees a V which is not finite is NaN
                            const uint32_t* seen = C.bad[wg][(cleans + 2) % 3];
                            uint32_t hit = 0;
                            if (STACKED) {
                                hit = __ballot_sync(0xffffffffu, ((vis[0] & seen[2 * (lane >> 4)]) | (vis[1] & seen[2 * (lane >> 4) + 1])) != 0);
                                hit |= hit >> 16;          // bit per row
                                if ((hit >> (lane >> 2)) & 1) sum = NAN;
                                if ((hit >> (8 + (lane >> 2))) & 1) sum1 = NAN;
                            } else if (valid) {
#pragma unroll 1
                                for (int w = 0; w < 4; w++) hit |= seen[w] ? seen[w] & tree_bits(a, g.s, mask, mask0, kb + 32 * w) : 0u;
                                if (hit) sum = NAN;
                            }
                        }
                    }
                    if (k) ok = __all_sync(0xffffffffu, mbar_wait(&C.x_free[wg], (k - 1) & 1, &g_tree_error));
                    if (!ok) break;
                    if (!STACKED) C.x[wg][tid] = make_float2(m, sum);
                    else if ((lane & 3) == 0) {
                        C.x[wg][r0] = make_float2(m, sum);
                        C.x[wg][r1] = make_float2(m1, sum1);
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&C.p_full[wg]);
                }
            } while (ok && seg_next<TW_ROWS, TW_KEYS>(a, g));
        }
    } else {
        // ---------------- the running output (thread = row, or half of it) ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(tw_regs_out(STACKED)));
        const int quad = warp & 3, r = STACKED ? quad * 16 + (lane & 15) : quad * 32 + lane;
        const uint32_t O = tmem + ((uint32_t)(quad * 32) << 16) + 256;
        int n = 0;
        if (N) {
            TreeSeg g = start.g;
            do {
                const bool valid = r < g.rows, live = quad * (STACKED ? 16 : 32) < g.rows;
                const bool first = g.tile0 == 0;
                uint64_t acc[64];
#pragma unroll
                for (int i = 0; i < 64; i++) acc[i] = 0;
                float M = -INFINITY, L = 0.0f;
                for (int t = 0; t < g.tiles && ok; t++, n++) {
                    const int b = (int)(n & 1);
                    const uint32_t k = (uint32_t)(n >> 1);
                    ok = __all_sync(0xffffffffu, mbar_wait(&C.o_full[b], k & 1, &g_tree_error));
                    if (!ok) break;
                    tc_fence_after();
                    const float2 x = C.x[b][r];
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&C.x_free[b]);
                    if (live) {
                        // a tile that the row sees nothing of (m = -inf, sum 0) has the weight 0
                        const bool up = valid && x.x > M;
                        if (__any_sync(0xffffffffu, up)) {
                            const float f = up ? ex2(M - x.x) : 1.0f;   // M = -inf: 0, all it scales is 0
                            const uint64_t f2 = pack2(f, f);
                            if (up) M = x.x;
                            L *= f;
#pragma unroll
                            for (int i = 0; i < 64; i++) acc[i] = fma2(acc[i], f2, 0ull);
                        }
                        const float w = x.x == -INFINITY ? 0.0f : ex2(x.x - M);
                        const uint64_t w2 = pack2(w, w);
                        L += x.y * w;
#pragma unroll
                        for (int q = 0; q < 8; q++) {
                            uint32_t o[16];
                            tmem_ld16(O + b * 128 + 16 * q, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 8; i++)
                                acc[8 * q + i] = fma2(pack2(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])), w2, acc[8 * q + i]);
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&C.o_free[b]);
                }
                if (!ok) break;
                const bool whole = g.tile0 == 0 && g.tiles == g.s.tiles;
                // stacked: lane i ends with the sums of the first 64 dims, lane i + 16 with those of the last
                constexpr int N2 = STACKED ? 32 : 64;
                const int side = STACKED ? lane >> 4 : 0;
                if (STACKED && live) {
#pragma unroll
                    for (int i = 0; i < 32; i++) {
                        const uint64_t other = __shfl_xor_sync(0xffffffffu, side ? acc[i] : acc[i + 32], 16);
                        acc[i] = add2(side ? acc[i + 32] : acc[i], other);
                    }
                }
                if (valid) {
                    const int R = g.rt * TW_ROWS + r;
                    const size_t part = ((size_t)blockIdx.x * 2 + (first ? 1 : 0)) * a.part_rows + r;
                    float* dst = a.part_o + part * HD;
                    float f = 1.0f;
                    if (whole) {
                        dst = a.out + ((int64_t)(g.s.s0 + R / a.nrep) * a.hq + g.kvh * a.nrep + R % a.nrep) * HD;
                        f = L != 0.0f ? 1.0f / L : 0.0f;
                    } else if (side == 0) {
                        *(float2*)(a.part_ml + part * 2) = make_float2(M, L);
                    }
                    dst += side * 64;
                    const uint64_t f2 = pack2(f, f);
#pragma unroll
                    for (int i = 0; i < N2; i += 2) {
                        float4 y;
                        unpack2(fma2(acc[i], f2, 0ull), y.x, y.y);
                        unpack2(fma2(acc[i + 1], f2, 0ull), y.z, y.w);
                        *(float4*)(dst + 2 * i) = y;
                    }
                }
                if (!whole && first && threadIdx.x == 12 * 32) {
                    const int64_t end = start.u0 + n - g.tiles + g.s.tiles;
                    int lo = blockIdx.x, hi = a.G;   // the CTA that has the item's last unit
                    while (hi - lo > 1) {
                        const int mid = (lo + hi) / 2;
                        if (a.bounds[mid] < end) lo = mid;
                        else hi = mid;
                    }
                    a.cuts[blockIdx.x] = {g.rows, g.s.s0, g.rt * TW_ROWS, g.kvh, lo - (int)blockIdx.x + 1};
                }
            } while (seg_next<TW_ROWS, TW_KEYS>(a, g));
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// ------------------------------------------------------------------------------------------
// tree_few_kernel<MT>: up to 16 MT rows per kv head (a chain of drafts, a small tree), mma.sync.
// With so few rows the K/V bytes are all that counts, and a warp that owns whole blocks of 16 keys has
// no hand-over to wait for: one CTA (3 consumer warps, 1 TMA producer warp, 2 CTAs per SM) per
// (sequence, kv head, split of its blocks), consumer warp w takes blocks w, w + 3, ... from a ring of
// whole blocks.  Per block: S = Q K^T and P V on m16n8k16, q and p as fp16 halves (hi + lo) as in the
// wide kernel; a block's P V starts from zero and is added to the running output in fp32 rounded to
// nearest, because the tensor core cuts its sums off.  The warps merge in shared memory; splits leave
// their parts for tree_join_kernel.
// What bounds it: latency while contexts are short (8 tokens x 200: 7.9 us), HBM when they are long (8 x
// 100,003: 71 us, 5.8 TB/s).
// ------------------------------------------------------------------------------------------
constexpr int TF_CONS = 3;
constexpr int TF_STAGES = 9;
// A slot always belongs to the same consumer warp: one that another warp had not emptied yet would look
// full by the parity of its phase.
static_assert(TF_STAGES % TF_CONS == 0, "ring and consumers");
constexpr int TF_TILE = KVB * HD * 2;             // 4 KB: [half of 64 dims][16 keys][128 B]
constexpr int TF_STAGE = 2 * TF_TILE;             // K, V

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr));
}
__device__ __forceinline__ void mma_h(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// byte address of 16-byte chunk c (of 16) of row r in a swizzled tile
__device__ __forceinline__ uint32_t tf_at(uint32_t tile, int r, int c) {
    return tile + (uint32_t)(c >> 3) * (TF_TILE / 2) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

template <int MT>
__global__ void __launch_bounds__((TF_CONS + 1) * 32, 2) tree_few_kernel(
    const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const TreeArgs a, int bps, int splits) {
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* ring = smem;
    uint4* qf = (uint4*)(smem + TF_STAGES * TF_STAGE);            // [MT][k-step][hi, lo][lane]
    uint64_t* full = (uint64_t*)(qf + MT * 8 * 2 * 32);
    uint64_t* empty = full + TF_STAGES;
    float* wm = (float*)(empty + TF_STAGES);                       // [warp][row]
    float* wl = wm + TF_CONS * 16 * MT;
    float* qc = wl + TF_CONS * 16 * MT;                            // [row] scale of the scores, in powers of 2
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int gid = lane >> 2, tig = lane & 3;
    if (smem_u32(smem) & 1023) {                  // the swizzled tiles would not match their addresses
        if (threadIdx.x == 0) atomicExch(&g_tree_error, DCG_DEVERR_TIMEOUT);
        return;
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < TF_STAGES; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        fence_mbar_init();
    }
    pdl_wait();
    const int seq = blockIdx.x / a.hkv, kvh = blockIdx.x % a.hkv;
    const TreeSeq s = tree_seq<16 * MT, KVB>(a, seq, kvh == 0 && blockIdx.y == 0);
    const int rows = s.ns * a.nrep, hist = s.L - s.ns;
    const int b0 = blockIdx.y * bps, nb = max(0, min(s.tiles, b0 + bps) - b0);
    if (rows == 0) return;                        // no drafted tokens, or a sequence that is out of range
    // Q as A fragments: k-step j holds dims 16 j .. +15; rows gid (a0, a2) and gid + 8 (a1, a3).  Warp w
    // makes row tile w.
    if (warp < MT) {
        const float* q[2];
        float2 x[2][16];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int r = min(16 * warp + gid + 8 * h, rows - 1);
            q[h] = a.q + ((int64_t)(s.s0 + r / a.nrep) * a.hq + kvh * a.nrep + r % a.nrep) * HD + 2 * tig;
#pragma unroll
            for (int j = 0; j < 16; j++) x[h][j] = *(const float2*)(q[h] + 8 * j);
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float m = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; j++) m = fmaxf(m, fmaxf(fabsf(x[h][j].x), fabsf(x[h][j].y)));
            uint32_t u = __float_as_uint(m);      // also of NaN and infinities, which make the row NaN
            u = max(u, __shfl_xor_sync(0xffffffffu, u, 1));
            u = max(u, __shfl_xor_sync(0xffffffffu, u, 2));
            int e = (int)(u >> 23) - 127;
            e = e < -100 ? -100 : e > 120 ? 120 : e;
            const float f = copysignf(__uint_as_float((uint32_t)(127 - e) << 23), a.scale_log2);
            if (tig == 0) qc[16 * warp + gid + 8 * h] = fmaxf(fabsf(a.scale_log2) * __uint_as_float((uint32_t)(127 + e) << 23), 1e-37f);
#pragma unroll
            for (int j = 0; j < 16; j++) {
                x[h][j].x *= f;
                x[h][j].y *= f;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            uint4 hi, lo;
            cut_h2(x[0][2 * j].x, x[0][2 * j].y, hi.x, lo.x);
            cut_h2(x[1][2 * j].x, x[1][2 * j].y, hi.y, lo.y);
            cut_h2(x[0][2 * j + 1].x, x[0][2 * j + 1].y, hi.z, lo.z);
            cut_h2(x[1][2 * j + 1].x, x[1][2 * j + 1].y, hi.w, lo.w);
            qf[((warp * 8 + j) * 2) * 32 + lane] = hi;
            qf[((warp * 8 + j) * 2 + 1) * 32 + lane] = lo;
        }
    }
    __syncthreads();

    bool ok = true;
    float o[MT][16][4];                           // [row tile][8 dims][rows gid (0, 1) and gid + 8 (2, 3)]
    float m[MT][2], l[MT][2];
    uint32_t poison = 0;
#pragma unroll
    for (int t = 0; t < MT; t++) {
#pragma unroll
        for (int n = 0; n < 16; n++) o[t][n][0] = o[t][n][1] = o[t][n][2] = o[t][n][3] = 0.0f;
        m[t][0] = m[t][1] = -INFINITY;
        l[t][0] = l[t][1] = 0.0f;
    }
    if (warp == TF_CONS) {
        if (lane == 0) {
            const int beyond = (int)(a.n_arena_blocks * a.n_layer * KVB);   // out of the arena: zeros
            const int* bt = a.bt + (int64_t)seq * a.mbs + b0;
            int next = nb ? bt[0] : 0, i = 0;
            for (; i < nb; i++) {
                const int st = i % TF_STAGES, b = next;
                if (i + 1 < nb) next = bt[i + 1];
                const bool in = b >= 0 && b < a.n_arena_blocks;
                if (!in) atomicExch(&g_tree_error, DCG_DEVERR_INDEX);
                const int row = in ? (b * a.n_layer + a.layer) * KVB : beyond;
                if (i >= TF_STAGES) ok = mbar_wait(&empty[st], (uint32_t)((i / TF_STAGES - 1) & 1), &g_tree_error);
                if (!ok) break;
                mbar_arrive_expect_tx(&full[st], TF_STAGE);
                tma_load_4d(ring + (size_t)st * TF_STAGE, &kmap, 0, row, 0, kvh, &full[st]);
                tma_load_4d(ring + (size_t)st * TF_STAGE + TF_TILE, &vmap, 0, row, 0, kvh, &full[st]);
            }
            if (!ok)                               // given up: the copies in flight land before the CTA ends
                for (int x = max(0, i - TF_STAGES); x < i; x++) mbar_wait(&full[x % TF_STAGES], (uint32_t)((x / TF_STAGES) & 1), &g_tree_error, 1u << 16);
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
    } else {
        const uint32_t ring_s = smem_u32(ring);
        const int mi = lane >> 3, mr = lane & 7;  // ldmatrix: matrix, row in it
        float c[MT][2];
        int tok[MT][2];
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                c[t][h] = qc[16 * t + gid + 8 * h];
                tok[t][h] = s.s0 + min(16 * t + gid + 8 * h, rows - 1) / a.nrep;
            }
        for (int i = warp; i < nb; i += TF_CONS) {
            const int st = i % TF_STAGES;
            ok = __all_sync(0xffffffffu, mbar_wait(&full[st], (uint32_t)((i / TF_STAGES) & 1), &g_tree_error));
            if (!ok) break;
            const uint32_t kt = ring_s + (uint32_t)st * TF_STAGE, vt = kt + TF_TILE;
            const int kb = (b0 + i) * KVB;
            // ---- S: lane has rows gid, gid + 8 and keys 8 n + 2 tig, + 1 ----
            float sh[MT][2][4], sl[MT][2][4];
#pragma unroll
            for (int t = 0; t < MT; t++)
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sh[t][n][e] = sl[t][n][e] = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                uint32_t k0, k1, k2, k3;
                ldsm_x4(tf_at(kt, (mi >> 1) * 8 + mr, 2 * j + (mi & 1)), k0, k1, k2, k3);
#pragma unroll
                for (int t = 0; t < MT; t++) {
                    const uint4 hi = qf[((t * 8 + j) * 2) * 32 + lane], lo = qf[((t * 8 + j) * 2 + 1) * 32 + lane];
                    mma_h(sh[t][0], hi, k0, k1);
                    mma_h(sl[t][0], lo, k0, k1);
                    mma_h(sh[t][1], hi, k2, k3);
                    mma_h(sl[t][1], lo, k2, k3);
                }
            }
            // ---- masks, and V that must not reach the sums ----
            uint32_t vm01 = 0xFFFFFFFFu, vm23 = 0xFFFFFFFFu;   // V of keys 2 tig, +1 and 8 + 2 tig, +1
            uint32_t vis[MT][2];
            const bool special = kb + KVB > hist;
            if (special) {
                // V of slots past the context may be anything, and that of a drafted token that a row does
                // not see may be NaN: 0 x NaN is NaN, so such V count as zeros
                bool odd = false;
                const int key = kb + (lane >> 1);
                if (key >= hist && key < s.L) {
                    const uint32_t v = vt + (lane & 1) * (TF_TILE / 2) + (lane >> 1) * 128;
#pragma unroll
                    for (int x = 0; x < 8; x++) {
                        uint32_t y[4];
                        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(y[0]), "=r"(y[1]), "=r"(y[2]), "=r"(y[3]) : "r"(v + ((x + lane) & 7) * 16));
#pragma unroll
                        for (int e = 0; e < 4; e++) odd |= (y[e] & 0x7C00u) == 0x7C00u || (y[e] & 0x7C000000u) == 0x7C000000u;
                    }
                }
                const uint32_t odds = __ballot_sync(0xffffffffu, odd);
                uint32_t bad = 0;                  // bit per key
#pragma unroll
                for (int x = 0; x < KVB; x++) bad |= ((odds >> (2 * x)) & 3u ? 1u : 0u) << x;
                const int n = s.L - kb;
                const uint32_t none = bad | (n >= KVB ? 0u : 0xFFFFu << n);
                vm01 = ((none >> (2 * tig)) & 1 ? 0u : 0x0000FFFFu) | ((none >> (2 * tig + 1)) & 1 ? 0u : 0xFFFF0000u);
                vm23 = ((none >> (8 + 2 * tig)) & 1 ? 0u : 0x0000FFFFu) | ((none >> (9 + 2 * tig)) & 1 ? 0u : 0xFFFF0000u);
#pragma unroll
                for (int t = 0; t < MT; t++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint64_t* m = (const uint64_t*)a.mask + (int64_t)tok[t][h] * a.words;
                        vis[t][h] = tree_bits(a, s, m, *m, kb);
                        if (vis[t][h] & bad) poison |= 1u << (2 * t + h);
                    }
            }
            // ---- p, and its halves as A fragments ----
            uint4 ph[MT], pl[MT];
            float corr[MT][2];
#pragma unroll
            for (int t = 0; t < MT; t++) {
                float p[2][4];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float mx = -INFINITY;
#pragma unroll
                    for (int n = 0; n < 2; n++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            float v = sh[t][n][2 * h + e] + sl[t][n][2 * h + e];
                            if (special && !((vis[t][h] >> (8 * n + 2 * tig + e)) & 1)) v = -INFINITY;
                            p[n][2 * h + e] = v;
                            mx = fmaxf(mx, v);
                        }
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    const float mn = fmaxf(m[t][h], mx * c[t][h]);
                    corr[t][h] = mn == -INFINITY ? 1.0f : ex2(m[t][h] - mn);
                    m[t][h] = mn;
                    const float shift = TW_SHIFT - (mn == -INFINITY ? 0.0f : mn);
                    float sum = 0.0f;
#pragma unroll
                    for (int n = 0; n < 2; n++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            p[n][2 * h + e] = ex2(fmaf(p[n][2 * h + e], c[t][h], shift));
                            sum += p[n][2 * h + e];
                        }
                    l[t][h] = l[t][h] * corr[t][h] + sum;   // this lane's four keys; the lanes are joined at the end
                }
                cut_h2(p[0][0], p[0][1], ph[t].x, pl[t].x);
                cut_h2(p[0][2], p[0][3], ph[t].y, pl[t].y);
                cut_h2(p[1][0], p[1][1], ph[t].z, pl[t].z);
                cut_h2(p[1][2], p[1][3], ph[t].w, pl[t].w);
            }
            // ---- O = O corr + P V ----
#pragma unroll
            for (int n2 = 0; n2 < 8; n2++) {
                uint32_t v0, v1, v2, v3;
                ldsm_x4_t(tf_at(vt, (mi & 1) * 8 + mr, 2 * n2 + (mi >> 1)), v0, v1, v2, v3);
                v0 &= vm01;
                v2 &= vm01;
                v1 &= vm23;
                v3 &= vm23;
#pragma unroll
                for (int t = 0; t < MT; t++) {
                    float y0[4] = {0.f, 0.f, 0.f, 0.f}, y1[4] = {0.f, 0.f, 0.f, 0.f};
                    mma_h(y0, pl[t], v0, v1);
                    mma_h(y1, pl[t], v2, v3);
                    mma_h(y0, ph[t], v0, v1);
                    mma_h(y1, ph[t], v2, v3);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        o[t][2 * n2][e] = fmaf(o[t][2 * n2][e], corr[t][e >> 1], y0[e]);
                        o[t][2 * n2 + 1][e] = fmaf(o[t][2 * n2 + 1][e], corr[t][e >> 1], y1[e]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
        }
    }
    pdl_trigger();
    ok = __syncthreads_and(ok);
    if (!ok) return;
    // ---- merge the consumer warps: the ring becomes [warp][row][dim] ----
    float* acc = (float*)ring;
    static_assert(TF_CONS * 16 * MT * HD * 4 <= TF_STAGES * TF_STAGE, "merge space");
    if (warp < TF_CONS) {
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int r = 16 * t + gid + 8 * h;
                float x = l[t][h];
                x += __shfl_xor_sync(0xffffffffu, x, 1);
                x += __shfl_xor_sync(0xffffffffu, x, 2);
                if ((poison >> (2 * t + h)) & 1) x = NAN;
                if (tig == 0) {
                    wm[warp * 16 * MT + r] = m[t][h];
                    wl[warp * 16 * MT + r] = x;
                }
#pragma unroll
                for (int n = 0; n < 16; n++)
                    *(float2*)&acc[(warp * 16 * MT + r) * HD + 8 * n + 2 * tig] = make_float2(o[t][n][2 * h], o[t][n][2 * h + 1]);
            }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < rows * (HD / 4); x += (TF_CONS + 1) * 32) {
        const int r = x / (HD / 4), d = x % (HD / 4) * 4;
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int w = 0; w < TF_CONS; w++) M = fmaxf(M, wm[w * 16 * MT + r]);
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < TF_CONS; w++) {
            const float lw = wl[w * 16 * MT + r], f = lw != 0.0f ? ex2(wm[w * 16 * MT + r] - M) : 0.0f;
            if (lw == 0.0f) continue;
            const float4 z = *(const float4*)&acc[(w * 16 * MT + r) * HD + d];
            L += lw * f;
            y.x += z.x * f;
            y.y += z.y * f;
            y.z += z.z * f;
            y.w += z.w * f;
        }
        if (splits == 1) {
            const float inv = L != 0.0f ? 1.0f / L : 0.0f;
            *(float4*)(a.out + ((int64_t)(s.s0 + r / a.nrep) * a.hq + kvh * a.nrep + r % a.nrep) * HD + d) =
                make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
        } else {
            const size_t part = ((size_t)blockIdx.x * splits + blockIdx.y) * a.part_rows + r;
            *(float4*)(a.part_o + part * HD + d) = y;
            if (d == 0) *(float2*)(a.part_ml + part * 2) = make_float2(M, L);
        }
    }
}

// The parts of a row, 32 at a time: m and l a lane each, then the outputs with all loads apart from the
// sums (a lane 4 dims).  part(x): index of the x-th part.
// LOADS outputs are under way at a time: 16 where an item has many parts, 4 (and twice the warps) where few.
template <int LOADS, class F>
__device__ __forceinline__ void tree_join(const TreeArgs& a, int parts, F part, float* dst) {
    const int lane = threadIdx.x & 31;
    float M = -INFINITY, L = 0.0f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int x0 = 0; x0 < parts; x0 += 32) {
        const int n = min(32, parts - x0);
        const int p = lane < n ? (int)part(x0 + lane) : 0;
        float4 z[LOADS];
        auto load = [&](int i0) {
#pragma unroll
            for (int i = 0; i < LOADS; i++) {
                const int q = __shfl_sync(0xffffffffu, p, i0 + i);
                if (i0 + i < n) z[i] = *(const float4*)(a.part_o + (int64_t)q * HD + 4 * lane);
            }
        };
        load(0);                                   // beside the maxima
        float2 y = make_float2(-INFINITY, 0.0f);
        if (lane < n) y = *(const float2*)(a.part_ml + (int64_t)p * 2);
        float m = fmaxf(M, y.x);
#pragma unroll
        for (int i = 16; i; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
        const float f = M == -INFINITY ? 0.0f : ex2(M - m), w = y.y == 0.0f ? 0.0f : ex2(y.x - m);
        float l = y.y * w;
#pragma unroll
        for (int i = 16; i; i >>= 1) l += __shfl_xor_sync(0xffffffffu, l, i);
        M = m;
        L = L * f + l;
        o.x *= f;
        o.y *= f;
        o.z *= f;
        o.w *= f;
        const uint32_t used = __ballot_sync(0xffffffffu, y.y != 0.0f);   // the others' outputs were not written
        for (int i0 = 0; i0 < n; i0 += LOADS) {
            if (i0) load(i0);
#pragma unroll
            for (int i = 0; i < LOADS; i++) {
                const float v = __shfl_sync(0xffffffffu, w, i0 + i);
                if ((used >> (i0 + i)) & 1) {
                    o.x += z[i].x * v;
                    o.y += z[i].y * v;
                    o.z += z[i].z * v;
                    o.w += z[i].w * v;
                }
            }
        }
    }
    const float inv = L != 0.0f ? 1.0f / L : 0.0f;
    *(float4*)(dst + 4 * lane) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

// tree_few_kernel's splits: a warp per row, CTA (sequence and kv head, 8 rows)
constexpr int TC_ROWS = 8;
template <int LOADS>
__global__ void __launch_bounds__(TC_ROWS * 32) tree_join_kernel(const TreeArgs a, int splits) {
    pdl_wait();
    pdl_trigger();
    const int seq = blockIdx.x / a.hkv, kvh = blockIdx.x % a.hkv, r = blockIdx.y * TC_ROWS + (threadIdx.x >> 5);
    const TreeSeq s = tree_seq<TW_ROWS, TW_KEYS>(a, seq, false);
    if (r >= s.ns * a.nrep) return;
    tree_join<LOADS>(a, splits, [&](int x) { return ((int64_t)blockIdx.x * splits + x) * a.part_rows + r; },
              a.out + ((int64_t)(s.s0 + r / a.nrep) * a.hq + kvh * a.nrep + r % a.nrep) * HD);
}

// tree_wide_kernel's items that several CTAs worked on, in CTA order: CTA (CTA that began an item, 8 rows)
template <int LOADS>
__global__ void __launch_bounds__(TC_ROWS * 32) tree_combine_kernel(const TreeArgs a) {
    pdl_wait();
    pdl_trigger();
    const int c = blockIdx.x, r = blockIdx.y * TC_ROWS + (threadIdx.x >> 5);
    const TreeCut cut = a.cuts[c];
    if (r >= cut.rows) return;
    const int R = cut.row0 + r;
    tree_join<LOADS>(a, cut.parts,
              [&](int x) { return ((int64_t)(c + x) * 2 + (x == 0 ? 1 : 0)) * a.part_rows + r; },
              a.out + ((int64_t)(cut.s0 + R / a.nrep) * a.hq + cut.kvh * a.nrep + R % a.nrep) * HD);
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn();  // qmm.cu

// arena as (64 dims of a half, slot, half, kv head); one box: 16 slots of one half, or of both
static cudaError_t tree_map(CUtensorMap* map, const void* arena, int hkv, int64_t n_slots, int halves) {
    auto fn = encode_fn();
    if (!fn) return cudaErrorNotSupported;
    const cuuint64_t dims[4] = {64u, (cuuint64_t)n_slots, 2u, (cuuint64_t)hkv};
    const cuuint64_t strides[3] = {(cuuint64_t)hkv * HD * 2, 128u, (cuuint64_t)HD * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)KVB, (cuuint32_t)halves, 1};
    const cuuint32_t es[4] = {1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(arena), dims, strides, box, es,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? cudaSuccess
               : cudaErrorInvalidValue;
}

struct TreePlan {
    bool few;                   // tree_few_kernel
    int rows;                   // of a part
    int splits, bps;            // few: splits of a sequence's blocks, blocks of one
    int G, q_rows, row_tiles;   // wide
    size_t o_bytes, ml_bytes, cut_bytes, start_bytes, prefix_bytes, bound_bytes, q_bytes, e_bytes;
};
constexpr int TF_MIN = 6;
static TreePlan tree_plan(int n_seqs, int hq, int hkv, int max_seq_tokens, int max_ctx) {
    TreePlan p = {};
    const int64_t rows = (int64_t)max_seq_tokens * (hq / hkv);
    // few: a CTA for TF_MIN blocks at least, and all CTAs at once (two per SM).  Times in us of 1 / 4 / 16
    // sequences with 8 kv heads and 16 rows, this plan against decode attention's two waves: 1,000
    // tokens 7.6 / 10.3 / 19 against 14 / 14 / 30.
    const int nblk = max_ctx > KVB ? (max_ctx - 1) / KVB + 1 : 1;
    const int64_t fit = 2 * (int64_t)num_sms() / ((int64_t)n_seqs * hkv);
    p.splits = (int)min((int64_t)(nblk - 1) / TF_MIN + 1, max(fit, (int64_t)1));
    // no second launch (2.4 us of the host's time) for 16 blocks: 200 tokens 7.8 us against 7.1 in a graph,
    // 10.9 against 13.3 from Python; beyond 16 rows for 8
    if (nblk <= (rows <= 16 ? 16 : 8)) p.splits = 1;
    p.bps = (nblk - 1) / p.splits + 1;
    p.splits = (nblk - 1) / p.bps + 1;
    // Up to 16 rows few wins while its CTAs have up to 96 blocks, or as many each: 64 sequences of up to 1,024
    // tokens 45 against wide's 53 us, of up to 4,096 140 against 117, one of 100,003 71 against 80.  Beyond 16
    // rows, up to 32 blocks: one sequence of 4,000 tokens 16.3 against 17.5, of 20,000 33.2 against 31.8.
    p.few = rows <= 16 ? p.bps <= 96 || n_seqs == 1 : rows <= 32 && p.bps <= 32;
    size_t parts;
    if (p.few) {
        p.rows = (int)rows;
        parts = p.splits > 1 ? (size_t)n_seqs * hkv * p.splits : 0;
    } else {
        p.G = min(num_sms(), TQ_WARPS * 32 - 1);               // a planning thread each
        p.rows = (int)(rows < TW_ROWS ? rows : TW_ROWS);
        p.q_rows = p.rows <= TW_STACK ? (p.rows + 15) / 16 * 16 : (p.rows + 7) / 8 * 8;
        p.row_tiles = (int)((rows + TW_ROWS - 1) / TW_ROWS);
        parts = (size_t)2 * p.G;
        p.cut_bytes = align256((size_t)p.G * sizeof(TreeCut));
        p.start_bytes = align256((size_t)p.G * sizeof(TreeStart));
        p.prefix_bytes = align256((size_t)n_seqs * 2 * 8);
        p.bound_bytes = align256((size_t)(p.G + 1) * 8);
        const size_t q = (size_t)n_seqs * p.row_tiles * hkv * p.q_rows;
        p.q_bytes = align256(q * 512);
        p.e_bytes = align256(q);
    }
    p.o_bytes = align256(parts * p.rows * HD * 4);
    p.ml_bytes = align256(parts * p.rows * 2 * 4);
    return p;
}
size_t tree_scratch_bytes(int n_seqs, int hq, int hkv, int max_seq_tokens, int max_ctx) {
    const TreePlan p = tree_plan(n_seqs, hq, hkv, max_seq_tokens, max_ctx);
    return p.o_bytes + p.ml_bytes + p.cut_bytes + p.start_bytes + p.prefix_bytes + p.bound_bytes + p.q_bytes + p.e_bytes;
}

template <int MT>
static cudaError_t launch_few(const CUtensorMap& km, const CUtensorMap& vm, const TreeArgs& a, const TreePlan& p, cudaStream_t st) {
    const size_t smem = (size_t)TF_STAGES * TF_STAGE + MT * 8 * 2 * 32 * 16 + 2 * TF_STAGES * 8 + (2 * TF_CONS + 1) * 16 * MT * 4;
    cudaError_t e = DCG_SMEM_ATTR(tree_few_kernel<MT>, smem);
    if (e != cudaSuccess) return e;
    e = launch_pdl(tree_few_kernel<MT>, dim3((unsigned)(a.n_seqs * a.hkv), (unsigned)p.splits), dim3((TF_CONS + 1) * 32), smem,
                   st, km, vm, a, p.bps, p.splits);
    if (e != cudaSuccess || p.splits == 1) return e;
    return launch_pdl(p.splits > 8 ? tree_join_kernel<16> : tree_join_kernel<4>, dim3((unsigned)(a.n_seqs * a.hkv), (unsigned)((p.rows + TC_ROWS - 1) / TC_ROWS)),
                      dim3(TC_ROWS * 32), 0, st, a, p.splits);
}

cudaError_t launch_paged_attn_tree(const float* q, const void* karena, const void* varena, int64_t n_arena_blocks,
                                   int n_layer, int layer, const int* bt, int mbs, const int* seq_starts,
                                   const int* ctx, const int64_t* mask, int words, int n_tok, int n_seqs,
                                   int max_seq_tokens, int hq, int hkv, int max_ctx, float scale, float* out,
                                   void* scratch, cudaStream_t st) {
    const TreePlan p = tree_plan(n_seqs, hq, hkv, max_seq_tokens, max_ctx);
    TreeArgs a;
    a.q = q;
    a.n_arena_blocks = n_arena_blocks;
    a.n_layer = n_layer; a.layer = layer; a.bt = bt; a.mbs = mbs; a.starts = seq_starts; a.ctx = ctx;
    a.mask = mask; a.words = words; a.n_tok = n_tok; a.n_seqs = n_seqs; a.max_tok = max_seq_tokens; a.max_ctx = max_ctx;
    a.hq = hq; a.hkv = hkv; a.nrep = hq / hkv;
    a.scale_log2 = scale * LOG2E;
    a.out = out;
    uint8_t* at = (uint8_t*)scratch;
    a.part_o = (float*)at;
    a.part_ml = (float*)(at += p.o_bytes);
    a.cuts = (TreeCut*)(at += p.ml_bytes);
    a.begins = (TreeStart*)(at += p.cut_bytes);
    a.prefix = (int64_t*)(at += p.start_bytes);
    a.G = p.G;
    a.bounds = (int64_t*)(at += p.prefix_bytes);
    a.q_tiles = at += p.bound_bytes;
    a.q_exps = (int8_t*)(at += p.q_bytes);
    a.part_rows = p.rows;
    a.q_rows = p.q_rows;
    a.row_tiles = p.row_tiles;
    CUtensorMap km, vm;
    const int64_t n_slots = n_arena_blocks * n_layer * KVB;
    cudaError_t e = tree_map(&km, karena, hkv, n_slots, p.few ? 2 : 1);
    if (e == cudaSuccess) e = tree_map(&vm, varena, hkv, n_slots, p.few ? 2 : 1);
    if (e != cudaSuccess) return e;
    if (p.few) return p.rows <= 16 ? launch_few<1>(km, vm, a, p, st) : launch_few<2>(km, vm, a, p, st);
    const bool stacked = p.rows <= TW_STACK;
    e = stacked ? DCG_SMEM_ATTR(tree_wide_kernel<true>, TW_SMEM) : DCG_SMEM_ATTR(tree_wide_kernel<false>, TW_SMEM);
    if (e != cudaSuccess) return e;
    // tokens with those behind a sequence's last whose rows belong to its last tile
    const int64_t q_tokens = ((int64_t)(p.row_tiles - 1) * TW_ROWS + p.q_rows + a.nrep - 1) / a.nrep;
    e = launch_pdl(tree_q_kernel, dim3((unsigned)((q_tokens * hq + TQ_ROWS - 1) / TQ_ROWS), (unsigned)n_seqs + 1), dim3(TQ_WARPS * 32), 0, st, a);
    if (e != cudaSuccess) return e;
    e = launch_pdl(stacked ? tree_wide_kernel<true> : tree_wide_kernel<false>, dim3((unsigned)p.G), dim3(TW_THREADS), (size_t)TW_SMEM, st, km, vm, a);
    if (e != cudaSuccess) return e;
    const int64_t items = (int64_t)n_seqs * p.row_tiles * hkv;   // at most
    return launch_pdl(items * 8 <= p.G ? tree_combine_kernel<16> : tree_combine_kernel<4>, dim3((unsigned)p.G, (unsigned)((p.rows + TC_ROWS - 1) / TC_ROWS)),
                      dim3(TC_ROWS * 32), 0, st, a);
}

}  // namespace dcg
