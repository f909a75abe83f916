// kv_pages.cu -- pages of the paged KV cache under sequences that branch: forking rows of a block
// table with reference counts and copy-on-write, and moving an accepted path's slots together.
//
// The reference's ref-counted BlockManager shares and copies blocks on the host
// (core/src/kv_cache.cpp:67-315); here the whole batch is planned and copied on the device, so a
// step can fork without waiting for the host.
#include "../../include/dcgpu.h"
#include "common.cuh"
#include "kernels.h"

namespace dcg {

constexpr int KVB = 16;   // tokens per page

__device__ int g_pages_error = 0;

cudaError_t pages_device_error(int* out, bool clear) {
    cudaError_t e = cudaMemcpyFromSymbol(out, g_pages_error, sizeof(int));
    if (e == cudaSuccess && clear && *out) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_pages_error, &zero, sizeof(int));
    }
    return e;
}

// ------------------------------------------------------------------------------------------
// kv_fork.  Row i of the table becomes a child of row p = parents[i]:
//   old rows drop their references, new rows take the first ceil(len_p / 16) pages of their parent;
//   in row order, a row whose last page is partly filled and has another holder asks for a page to
//   copy it to, and every row asks for the pages that len_p + reserve tokens need; request r gets
//   the r-th lowest page without a reference.
// A page that is copied from keeps a reference and a page that is copied to had none, so no copy
// reads what another writes.  Three launches (two for small tables), in stream order:
//   deltas  one CTA per old row p: ref[b] += kids(p) - 1 for its pages (0 for the usual single
//           child: no traffic), kids counted from `parents`; tables of up to FORK_SMALL entries leave
//           this to the plan's CTA, a launch less;
//   plan    one CTA: requests, their prefix sum, the scan for free pages, the rows' new lengths;
//   apply   column strips of the table permuted through shared memory (every row's old entry is read
//           before a new one is written), and the partial pages' slots copied.
// When the plan finds bad input or too few pages, apply takes the deltas back and nothing changes.
// What bounds it: the copied slots (HBM), behind the plan's chain of loads and scans in one CTA (6 us);
// a batch with few copies is that and the launches' latency.  8 rows, 28 layers: 9.6 us; 64 rows of
// beam search, 36 layers, 73 MB read and written: 22.7 us (the copies alone 11).
// ------------------------------------------------------------------------------------------
constexpr int FORK_MAX_ROWS = 4096;
constexpr int FORK_THREADS = 256;
constexpr int FORK_BATCH = 8;            // 16-byte loads in flight per thread of a copy (64 rows: 23.3 us; 4 or 16: 26.5)
constexpr int PLAN_THREADS = 1024;
constexpr int FORK_SMALL = 65536;        // table entries a CTA counts itself (8 rows 10.2 us where three launches took 12.1)
constexpr int PLAN_PER = 16;             // reference counts per thread and scan step
constexpr int STRIP_INTS = 8192;         // 32 KB of table entries per strip

struct ForkArgs {
    uint8_t *k, *v;
    int64_t n_pages_arena;
    int n_layer;
    int64_t slot_bytes;                  // one token's K (or V) of one layer
    int32_t* bt;
    int mbs;
    int32_t *lens, *held, *refs;
    const int32_t *parents, *reserve;
    int n, fill;
    int32_t* status;
    // scratch
    int32_t *bad;                        // [n] per old row, written by deltas
    int32_t *head;                       // {verdict, n_copies, columns}
    int32_t *new_len, *new_held, *old_held, *used, *src, *first, *copies;   // [n]
    int32_t* list;                       // pages handed out, by request
};

struct OldRow {
    int held, used, kids;
    bool bad;
};

// sizes of an old row with `kids` children (par: its own parent); a row that is bad moves nothing
__device__ __forceinline__ OldRow sized_row(const ForkArgs& a, int par, int64_t len, int held, int kids) {
    const int64_t used = (len + KVB - 1) / KVB;
    OldRow r;
    r.kids = kids;
    r.bad = held < 0 || held > a.mbs || par < -1 || par >= a.n || (kids && (len < 0 || used > held));
    r.held = r.bad ? 0 : held;
    r.used = r.bad ? 0 : (int)(used < 0 ? 0 : (used > held ? held : used));
    return r;
}
// the same with the children counted, by a CTA of FORK_THREADS
__device__ OldRow old_row(const ForkArgs& a, int p) {
    int kids = 0;
    for (int i0 = 0; i0 < a.n; i0 += FORK_THREADS) {
        const int i = i0 + threadIdx.x;
        kids += __syncthreads_count(i < a.n && a.parents[i] == p);
    }
    return sized_row(a, a.parents[p], a.lens[p], a.held[p], kids);
}

// ref[b] += sign * (kids - 1) for the pages that go to the children, -sign for the others, by threads
// first, first + step, ...; returns whether a page id was out of range
__device__ __forceinline__ bool add_deltas(const ForkArgs& a, int p, const OldRow& r, int sign, int first, int step) {
    bool bad = false;
    for (int j = first; j < r.held; j += step) {
        const int b = a.bt[(int64_t)p * a.mbs + j];
        const bool ok = b >= 0 && b < a.n_pages_arena;
        bad |= !ok;
        const int d = (j < r.used ? r.kids : 0) - 1;
        if (ok && d) atomicAdd(&a.refs[b], sign * d);
    }
    return bad;
}

__global__ void __launch_bounds__(FORK_THREADS) fork_deltas_kernel(const ForkArgs a) {
    pdl_wait();
    pdl_trigger();
    const int p = blockIdx.x;
    const OldRow r = old_row(a, p);
    const bool bad = add_deltas(a, p, r, 1, threadIdx.x, FORK_THREADS);
    const int any = __syncthreads_or(bad || r.bad);
    if (threadIdx.x == 0) a.bad[p] = any;
}

// exclusive prefix sum over the CTA's threads; total in *sum
__device__ int block_scan(int v, int* warp_sums, int* sum) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();   // the previous call's readers are done
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int w = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        warp_sums[lane] = w;
    }
    __syncthreads();
    *sum = warp_sums[31];
    return x - v + (warp ? warp_sums[warp - 1] : 0);
}

// SMALL: the deltas of all rows as well, a warp per row (n <= PLAN_THREADS: a thread per row elsewhere)
template <bool SMALL>
__global__ void __launch_bounds__(PLAN_THREADS) fork_plan_kernel(const ForkArgs a) {
    __shared__ int s_src[FORK_MAX_ROWS];     // partly filled last page of each new row, or -1
    // SMALL: read once, all loads together
    __shared__ int s_par[SMALL ? PLAN_THREADS : 1], s_len[SMALL ? PLAN_THREADS : 1], s_held[SMALL ? PLAN_THREADS : 1], s_kids[SMALL ? PLAN_THREADS : 1];
    __shared__ int warp_sums[32];
    __shared__ int s_copies;
    pdl_wait();
    pdl_trigger();
    const int t = threadIdx.x;
    if (t == 0) s_copies = 0;
    bool bad = false;
    int my_reserve = 0, my_now = 0, my_used = 0, my_held = 0;   // SMALL: of row t
    if (SMALL) {
        int p = -1;
        s_kids[t] = 0;
        if (t < a.n) {
            s_par[t] = p = a.parents[t];
            s_len[t] = a.lens[t];
            s_held[t] = my_held = a.held[t];
            my_reserve = a.reserve ? a.reserve[t] : 0;
            bad = p < -1 || p >= a.n;
        }
        __syncthreads();
        if (p >= 0 && !bad) atomicAdd(&s_kids[p], 1);
        __syncthreads();
        for (int r = t >> 5; r < a.n; r += PLAN_THREADS / 32) {
            const OldRow row = sized_row(a, s_par[r], s_len[r], s_held[r], s_kids[r]);
            bad |= row.bad;
            bad |= add_deltas(a, r, row, 1, t & 31, 32);
        }
    } else {
        for (int i = t; i < a.n; i += PLAN_THREADS) bad |= a.bad[i] != 0;
    }
    bad = __syncthreads_or(bad);
    if (bad) {
        if (t == 0) { a.head[0] = -1; *a.status = -1; }
        return;
    }
    // the new rows
    for (int i = t; i < a.n; i += PLAN_THREADS) {
        const int p = SMALL ? s_par[i] : a.parents[i];
        const int len = p < 0 ? 0 : SMALL ? s_len[p] : a.lens[p];
        const int more = SMALL ? my_reserve : a.reserve ? a.reserve[i] : 0;
        const int64_t need = p >= 0 ? (int64_t)len + more : 0;
        const int used = (len + KVB - 1) / KVB;
        const int64_t total = (need + KVB - 1) / KVB;
        bad |= p >= 0 && (more < 0 || total > a.mbs);
        s_src[i] = len % KVB ? a.bt[(int64_t)p * a.mbs + used - 1] : -1;
        a.new_len[i] = len;
        my_now = (int)(total > a.mbs ? a.mbs : total);
        my_used = used;
        if (!SMALL) my_held = a.held[i];
        a.new_held[i] = my_now;
        a.old_held[i] = my_held;
        a.used[i] = used;
    }
    bad = __syncthreads_or(bad);
    if (bad) {
        if (t == 0) { a.head[0] = -1; *a.status = -1; }
        return;
    }
    // requests, in row order (the copies' list in any order)
    int asked = 0, columns = 0;
    for (int i0 = 0; i0 < a.n; i0 += PLAN_THREADS) {
        const int i = i0 + t;
        int copy = 0, want = 0;
        if (i < a.n) {
            const int b = s_src[i];
            if (b >= 0) {
                const int held = __ldcg(&a.refs[b]);   // counts changed by this CTA's atomics: from L2
                int rank = 0;
                for (int j = 0; j < i; j++) rank += s_src[j] == b;
                copy = held - rank > 1;
            }
            const int now = SMALL ? my_now : a.new_held[i];
            want = copy + now - (SMALL ? my_used : a.used[i]);
            a.src[i] = copy ? b : -1;
            if (copy) a.copies[atomicAdd(&s_copies, 1)] = i;
            columns = max(columns, max(now, SMALL ? my_held : a.old_held[i]));
        }
        int sum;
        const int at = block_scan(want, warp_sums, &sum);
        if (i < a.n) a.first[i] = asked + at;
        asked += sum;
    }
    // the lowest pages without a reference
    const bool aligned = ((uintptr_t)a.refs & 15) == 0;
    int found = 0;
    for (int64_t b0 = 0; b0 < a.n_pages_arena && found < asked; b0 += PLAN_THREADS * PLAN_PER) {
        const int64_t b = b0 + (int64_t)t * PLAN_PER;
        uint32_t free_bits = 0;
        if (b + PLAN_PER <= a.n_pages_arena && aligned) {
#pragma unroll
            for (int u = 0; u < PLAN_PER; u += 4) {
                const int4 c = __ldcg((const int4*)(a.refs + b + u));
                free_bits |= ((c.x == 0) | (c.y == 0) << 1 | (c.z == 0) << 2 | (c.w == 0) << 3) << u;
            }
        } else {
#pragma unroll
            for (int u = 0; u < PLAN_PER; u++)
                if (b + u < a.n_pages_arena && __ldcg(&a.refs[b + u]) == 0) free_bits |= 1u << u;
        }
        int sum;
        int at = found + block_scan(__popc(free_bits), warp_sums, &sum);
        for (; free_bits; free_bits &= free_bits - 1, at++)
            if (at < asked) a.list[at] = (int)(b + __ffs(free_bits) - 1);
        found += sum;
    }
    for (int o = 16; o; o >>= 1) columns = max(columns, __shfl_xor_sync(0xffffffffu, columns, o));
    __syncthreads();   // list complete, every count read
    if ((t & 31) == 0) warp_sums[t >> 5] = columns;
    __syncthreads();
    if (found < asked) {
        if (t == 0) { a.head[0] = asked - found; *a.status = asked - found; }
        return;
    }
    for (int r = t; r < asked; r += PLAN_THREADS) a.refs[a.list[r]] = 1;
    for (int i = t; i < a.n; i += PLAN_THREADS)
        if (a.src[i] >= 0) atomicAdd(&a.refs[a.src[i]], -1);
    if (t == 0) {
        for (int w = 1; w < 32; w++) columns = max(columns, warp_sums[w]);
        a.head[0] = 0;
        a.head[1] = s_copies;
        a.head[2] = columns;
        *a.status = 0;
    }
}

// CTAs 0 .. strips-1: table columns; the rest: copies
__global__ void __launch_bounds__(FORK_THREADS) fork_apply_kernel(const ForkArgs a, int strips, int cols) {
    __shared__ int tile[STRIP_INTS];
    pdl_wait();
    pdl_trigger();
    if (a.head[0]) {   // nothing changes: the deltas are taken back
        for (int p = blockIdx.x; p < a.n; p += gridDim.x) {
            const OldRow r = old_row(a, p);
            add_deltas(a, p, r, -1, threadIdx.x, FORK_THREADS);
        }
        return;
    }
    if (blockIdx.x < strips) {
        const int j0 = blockIdx.x * cols;
        if (blockIdx.x == 0)
            for (int i = threadIdx.x; i < a.n; i += FORK_THREADS) {
                a.lens[i] = a.new_len[i];
                a.held[i] = a.new_held[i];
            }
        if (j0 >= a.head[2]) return;
        for (int e = threadIdx.x; e < a.n * cols; e += FORK_THREADS) {
            const int i = e / cols, j = j0 + e % cols;
            tile[e] = j < a.mbs ? a.bt[(int64_t)i * a.mbs + j] : 0;
        }
        __syncthreads();
        for (int e = threadIdx.x; e < a.n * cols; e += FORK_THREADS) {
            const int i = e / cols, j = j0 + e % cols;
            if (j >= a.mbs) continue;
            const int used = a.used[i], held = a.new_held[i], copy = a.src[i] >= 0;
            int b;
            if (j < used)
                b = copy && j == used - 1 ? a.list[a.first[i]] : tile[a.parents[i] * cols + e % cols];
            else if (j < held)
                b = a.list[a.first[i] + copy + j - used];
            else if (j < a.old_held[i])
                b = a.fill;
            else
                continue;
            a.bt[(int64_t)i * a.mbs + j] = b;
        }
        return;
    }
    // unit = (copy, layer, K or V): the page's first len % 16 slots are contiguous
    const int64_t units = (int64_t)a.head[1] * a.n_layer * 2;
    for (int64_t u = blockIdx.x - strips; u < units; u += gridDim.x - strips) {
        const int i = a.copies[u / (2 * a.n_layer)];
        const int layer = (int)(u / 2 % a.n_layer);
        uint8_t* arena = u & 1 ? a.v : a.k;
        const int64_t page_bytes = KVB * a.slot_bytes;
        const uint4* from = (const uint4*)(arena + ((int64_t)a.src[i] * a.n_layer + layer) * page_bytes);
        uint4* to = (uint4*)(arena + ((int64_t)a.list[a.first[i]] * a.n_layer + layer) * page_bytes);
        const int n16 = (int)(a.new_len[i] % KVB * a.slot_bytes / 16);
        // all of a thread's loads before its stores: from and to are different pages
        for (int x0 = threadIdx.x; x0 < n16; x0 += FORK_BATCH * FORK_THREADS) {
            uint4 r[FORK_BATCH];
#pragma unroll
            for (int e = 0; e < FORK_BATCH; e++)
                if (x0 + e * FORK_THREADS < n16) r[e] = __ldcs(from + x0 + e * FORK_THREADS);
#pragma unroll
            for (int e = 0; e < FORK_BATCH; e++)
                if (x0 + e * FORK_THREADS < n16) to[x0 + e * FORK_THREADS] = r[e];
        }
    }
}

static int64_t fork_list(int n, int mbs, int64_t n_arena_blocks) {
    const int64_t most = (int64_t)n * ((int64_t)mbs + 1);
    return most < n_arena_blocks ? most : n_arena_blocks;
}
size_t kv_fork_scratch_bytes(int n, int mbs, int64_t n_arena_blocks) {
    return align256((size_t)(n * (int64_t)8 + 4 + fork_list(n, mbs, n_arena_blocks)) * 4);
}

cudaError_t launch_kv_fork(void* k, void* v, int64_t n_arena_blocks, int n_layer, int64_t slot_bytes, int* bt,
                           int mbs, int* lens, int* held, int* refs, const int* parents, const int* reserve,
                           int n, int fill, int* status, void* scratch, cudaStream_t st) {
    ForkArgs a;
    a.k = (uint8_t*)k; a.v = (uint8_t*)v;
    a.n_pages_arena = n_arena_blocks; a.n_layer = n_layer; a.slot_bytes = slot_bytes;
    a.bt = bt; a.mbs = mbs; a.lens = lens; a.held = held; a.refs = refs;
    a.parents = parents; a.reserve = reserve; a.n = n; a.fill = fill; a.status = status;
    int* s = (int*)scratch;
    a.head = s; s += 4;
    a.bad = s; s += n;
    a.new_len = s; s += n;
    a.new_held = s; s += n;
    a.old_held = s; s += n;
    a.used = s; s += n;
    a.src = s; s += n;
    a.first = s; s += n;
    a.copies = s; s += n;
    a.list = s;
    cudaError_t e;
    if (n <= PLAN_THREADS && (int64_t)n * mbs <= FORK_SMALL) {
        e = launch_pdl(fork_plan_kernel<true>, dim3(1), dim3(PLAN_THREADS), 0, st, a);
    } else {
        e = launch_pdl(fork_deltas_kernel, dim3((unsigned)n), dim3(FORK_THREADS), 0, st, a);
        if (e != cudaSuccess) return e;
        e = launch_pdl(fork_plan_kernel<false>, dim3(1), dim3(PLAN_THREADS), 0, st, a);
    }
    if (e != cudaSuccess) return e;
    int cols = STRIP_INTS / n;
    cols = cols > 32 ? 32 : cols;
    const int strips = (mbs + cols - 1) / cols;
    return launch_pdl(fork_apply_kernel, dim3((unsigned)(strips + 4 * num_sms())), dim3(FORK_THREADS), 0, st, a,
                      strips, cols);
}
int kv_fork_max_rows() { return FORK_MAX_ROWS; }

// ------------------------------------------------------------------------------------------
// kv_compact.  For row s and every layer, slot base + path[j] goes to slot base + j, j ascending.
// path is strictly ascending, so path[j] >= j and a slot is read before or when it is written; each
// thread owns one 16-byte column of one layer's K or V for the whole path, so the order within a
// thread is the only order there is.  What bounds it: the moved bytes, 16 B loads with a batch of
// COMPACT_BATCH in flight per thread before the first store.  32 paths of 64 tokens, 36 layers (171 MB
// read and written): 31.1 us, 5.5 TB/s, of which the kernel's own 26 us are the rate of a copy; batches
// of 4 31.7, of 16 32.5.  One path of 8: 2.5 us, a launch.
// ------------------------------------------------------------------------------------------
constexpr int COMPACT_THREADS = 256;
constexpr int COMPACT_BATCH = 8;
constexpr int COMPACT_MAX_PATH = 1024;

__global__ void __launch_bounds__(COMPACT_THREADS) kv_compact_kernel(
    uint4* __restrict__ karena, uint4* __restrict__ varena, int64_t n_arena_blocks, int n_layer, int vecs,
    const int* __restrict__ bt, int mbs, const int* __restrict__ base_lens, const int* __restrict__ path,
    int max_path, const int* __restrict__ path_lens, int* __restrict__ ctx_lens) {
    extern __shared__ int64_t move[];        // {from, to} as page * n_layer * 16 + slot
    pdl_wait();
    pdl_trigger();
    const int s = blockIdx.y;
    const int base = base_lens[s], n = path_lens[s];
    bool bad = base < 0 || n < 0 || n > max_path || (int64_t)base + n > (int64_t)mbs * KVB;
    int skip = 0;                            // leading nodes that stay where they are
    if (!bad) {
        for (int j = threadIdx.x; j < n; j += COMPACT_THREADS) {
            const int at = path[(int64_t)s * max_path + j];
            const int before = j ? path[(int64_t)s * max_path + j - 1] : -1;
            const int64_t from = (int64_t)base + at, to = (int64_t)base + j;
            bool ok = at > before && at >= j && from < (int64_t)mbs * KVB;
            if (ok) {
                const int pf = bt[(int64_t)s * mbs + from / KVB], pt = bt[(int64_t)s * mbs + to / KVB];
                ok = pf >= 0 && pf < n_arena_blocks && pt >= 0 && pt < n_arena_blocks;
                move[2 * j] = (int64_t)pf * n_layer * KVB + from % KVB;
                move[2 * j + 1] = (int64_t)pt * n_layer * KVB + to % KVB;
            }
            bad |= !ok;
        }
    }
    bad = __syncthreads_or(bad);
    if (bad) {
        if (threadIdx.x == 0) atomicExch(&g_pages_error, DCG_DEVERR_INDEX);
        return;
    }
    while (skip < n && move[2 * skip] == move[2 * skip + 1]) skip++;
    if (blockIdx.x == 0 && threadIdx.x == 0) ctx_lens[s] = base + n;
    const int64_t item = (int64_t)blockIdx.x * COMPACT_THREADS + threadIdx.x;
    if (item >= (int64_t)2 * n_layer * vecs) return;
    const int x = (int)(item % vecs);
    const int layer = (int)(item / vecs % n_layer);
    uint4* arena = item >= (int64_t)n_layer * vecs ? varena : karena;
    arena += (int64_t)layer * KVB * vecs + x;
    for (int j0 = skip; j0 < n; j0 += COMPACT_BATCH) {
        uint4 r[COMPACT_BATCH];
#pragma unroll
        for (int u = 0; u < COMPACT_BATCH; u++)
            if (j0 + u < n) r[u] = arena[move[2 * (j0 + u)] * vecs];
#pragma unroll
        for (int u = 0; u < COMPACT_BATCH; u++)
            if (j0 + u < n) arena[move[2 * (j0 + u) + 1] * vecs] = r[u];
    }
}

cudaError_t launch_kv_compact(void* k, void* v, int64_t n_arena_blocks, int n_layer, int64_t slot_bytes,
                              const int* bt, int mbs, const int* base_lens, const int* path, int max_path,
                              const int* path_lens, int n_seqs, int* ctx_lens, cudaStream_t st) {
    const int vecs = (int)(slot_bytes / 16);
    const int64_t items = (int64_t)2 * n_layer * vecs;
    return launch_pdl(kv_compact_kernel, dim3((unsigned)((items + COMPACT_THREADS - 1) / COMPACT_THREADS), (unsigned)n_seqs),
                      dim3(COMPACT_THREADS), (size_t)max_path * 16, st, (uint4*)k, (uint4*)v, n_arena_blocks, n_layer,
                      vecs, bt, mbs, base_lens, path, max_path, path_lens, ctx_lens);
}
int kv_compact_max_path() { return COMPACT_MAX_PATH; }

}  // namespace dcg
