"""Torch-facing operators over libdcgpu.so.  torch only provides device memory and the current
stream; all arithmetic runs in the sm_100a kernels.  Names follow the reference operator surface:

  quantize_row_q8_0 / quantize_row_q8_K  ggml from_float (core/src/inference.cpp:887-894)
  mul_mat                                 smart_mul_mat / cb_gemv_custom / ggml_mul_mat on a
                                          quantized weight (inference.cpp:1043-1064, :840-948)
  QuantWeight                             a weight tensor resident on the device (the
                                          weight_tensor->data of cb_gemv_custom, uploaded once)
  HostContext                             the synchronous host-pointer boundary (dcg_ctx_*)
  paged_attn_tree                         the attention selector (inference.cpp:1506-1573) for drafted
                                          token trees, over the paged cache
  kv_fork / kv_compact                    BlockManager's shared, copied-on-write blocks
                                          (core/src/kv_cache.cpp:67-315), a batch at a time
  beam_select                             the k best continuations of groups of beams
"""
from __future__ import annotations

import ctypes

import numpy as np
import torch

from . import _lib
from .ggml_types import Q4_K, Q6_K, Q8_0, Q8_K, VEC_DOT_TYPE, block_size, row_size


def _stream(stream=None) -> int:
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def _ptr(t: torch.Tensor) -> int:
    return t.data_ptr()


def _check_cuda(t: torch.Tensor, name: str, dtype=None):
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")


def _quantize_rows(fn: str, qtype: int, x: torch.Tensor, out: torch.Tensor | None):
    _check_cuda(x, "x", torch.float32)
    k = x.shape[-1]
    m = x.numel() // k
    if out is None:
        out = torch.empty((m, row_size(qtype, k)), dtype=torch.uint8, device=x.device)
    _lib.check(getattr(_lib.load(), fn)(_ptr(x), _ptr(out), m, k, _stream()), fn)
    return out


def quantize_row_q8_0(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """f32 [..., k] -> ggml Q8_0 rows (uint8 [m, k/32*34])."""
    return _quantize_rows("dcg_quantize_row_q8_0", Q8_0, x, out)


def quantize_row_q8_K(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """f32 [..., k] -> ggml Q8_K rows (uint8 [m, k/256*292])."""
    return _quantize_rows("dcg_quantize_row_q8_K", Q8_K, x, out)


def quantize_weights(x: torch.Tensor, qtype: int) -> torch.Tensor:
    """Encode an f32 [n, k] weight as ggml Q8_0 / Q4_K / Q6_K rows on the device."""
    _check_cuda(x, "x", torch.float32)
    n, k = x.shape
    out = torch.empty((n, row_size(qtype, k)), dtype=torch.uint8, device=x.device)
    _lib.check(_lib.load().dcg_quantize_weights(qtype, _ptr(x), _ptr(out), n, k, _stream()),
               "dcg_quantize_weights")
    return out


class QuantWeight:
    """An n x k quantized weight in the device layout the matmul streams (dcg_weight_pack)."""

    def __init__(self, qtype: int, n: int, k: int, packed: torch.Tensor):
        self.qtype, self.n, self.k, self.packed = qtype, n, k, packed

    @classmethod
    def from_ggml(cls, rows: torch.Tensor, qtype: int, k: int) -> "QuantWeight":
        """rows: uint8 [n, >=row_size] ggml rows on the device (tensor nb[1] = rows.stride(0))."""
        _check_cuda(rows, "rows", torch.uint8)
        n = rows.shape[0]
        L = _lib.load()
        nbytes = L.dcg_packed_weight_size(qtype, n, k)
        if nbytes == 0:
            raise ValueError(f"unsupported weight type {qtype}")
        packed = torch.empty(nbytes, dtype=torch.uint8, device=rows.device)
        _lib.check(L.dcg_weight_pack(qtype, _ptr(rows), rows.stride(0), n, k, _ptr(packed),
                                     _stream()), "dcg_weight_pack")
        return cls(qtype, n, k, packed)

    @classmethod
    def from_float(cls, w: torch.Tensor, qtype: int) -> "QuantWeight":
        return cls.from_ggml(quantize_weights(w, qtype), qtype, w.shape[1])

    def to_ggml(self) -> torch.Tensor:
        rows = torch.empty((self.n, row_size(self.qtype, self.k)), dtype=torch.uint8,
                           device=self.packed.device)
        _lib.check(_lib.load().dcg_weight_unpack(self.qtype, _ptr(self.packed), self.n, self.k,
                                                 _ptr(rows), rows.stride(0), _stream()),
                   "dcg_weight_unpack")
        return rows

    @property
    def nbytes(self) -> int:
        """Algorithmic bytes (ggml block bytes) of the weight."""
        return self.n * row_size(self.qtype, self.k)


def mul_mat_scratch_size(qtype: int, n: int, k: int, m: int) -> int:
    return int(_lib.load().dcg_mul_mat_scratch_size(qtype, n, k, m))


def mul_mat_q_scratch_size(qtype: int, n: int, k: int, m: int) -> int:
    return int(_lib.load().dcg_mul_mat_q_scratch_size(qtype, n, k, m))


def mul_mat(w: QuantWeight, x: torch.Tensor, out: torch.Tensor | None = None,
            scratch: torch.Tensor | None = None) -> torch.Tensor:
    """y[m, n] = x[m, k] . W[n, k]^T with x quantized on the fly to W's vec_dot_type."""
    _check_cuda(x, "x", torch.float32)
    if x.shape[-1] != w.k:
        raise ValueError(f"x has k={x.shape[-1]}, weight has k={w.k}")
    m = x.numel() // w.k
    if out is None:
        out = torch.empty((m, w.n), dtype=torch.float32, device=x.device)
    need = mul_mat_scratch_size(w.qtype, w.n, w.k, m)
    if scratch is None:
        scratch = torch.empty(need, dtype=torch.uint8, device=x.device)
    _lib.check(_lib.load().dcg_mul_mat(w.qtype, _ptr(w.packed), w.n, w.k, _ptr(x), m, _ptr(out),
                                       _ptr(scratch), scratch.numel(), _stream()), "dcg_mul_mat")
    return out


def quantize_act(x: torch.Tensor, act_type: int, out: torch.Tensor | None = None) -> torch.Tensor:
    """f32 [m, k] -> device-layout activation (dcg_quantize_act) for mul_mat_q."""
    _check_cuda(x, "x", torch.float32)
    k = x.shape[-1]
    m = x.numel() // k
    L = _lib.load()
    if out is None:
        out = torch.empty(L.dcg_act_size(act_type, m, k), dtype=torch.uint8, device=x.device)
    _lib.check(L.dcg_quantize_act(act_type, _ptr(x), _ptr(out), m, k, _stream()), "dcg_quantize_act")
    return out


def mul_mat_q(w: QuantWeight, act: torch.Tensor, m: int, out: torch.Tensor | None = None,
              scratch: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """y[m, n] = W . act with act from quantize_act(x, VEC_DOT_TYPE[w.qtype])."""
    if out is None:
        out = torch.empty((m, w.n), dtype=torch.float32, device=act.device)
    if scratch is None:
        scratch = torch.zeros(max(1, mul_mat_q_scratch_size(w.qtype, w.n, w.k, m)),
                              dtype=torch.uint8, device=act.device)
    _lib.check(_lib.load().dcg_mul_mat_q(w.qtype, _ptr(w.packed), w.n, w.k, _ptr(act), m,
                                         _ptr(out), _ptr(scratch), scratch.numel(),
                                         _stream(stream)), "dcg_mul_mat_q")
    return out


def paged_attn_scratch_size(n_seqs: int, hq: int, hkv: int, max_ctx: int, head_dim: int = 128) -> int:
    return int(_lib.load().dcg_paged_attn_scratch_size(n_seqs, hq, hkv, head_dim, max_ctx))


def paged_attn_decode(q: torch.Tensor, k_arena: torch.Tensor, v_arena: torch.Tensor, n_layer: int,
                      layer: int, block_tables: torch.Tensor, ctx_lens: torch.Tensor, hkv: int,
                      max_ctx: int, scale: float | None = None, out: torch.Tensor | None = None,
                      scratch: torch.Tensor | None = None) -> torch.Tensor:
    """Decode attention of one query token per sequence over the paged fp16 KV arena.

    q [n_seqs, hq, 128] f32; k/v_arena fp16 (any shape, layout of dcgpu.h); block_tables
    [n_seqs, max_blocks] int32; ctx_lens [n_seqs] int32 (<= max_ctx)."""
    _check_cuda(q, "q", torch.float32)
    for t, nm in ((k_arena, "k_arena"), (v_arena, "v_arena")):
        _check_cuda(t, nm, torch.float16)
    _check_cuda(block_tables, "block_tables", torch.int32)
    _check_cuda(ctx_lens, "ctx_lens", torch.int32)
    n_seqs, hq, hd = q.shape
    if scale is None:
        scale = 1.0 / float(hd) ** 0.5
    if out is None:
        out = torch.empty_like(q)
    need = paged_attn_scratch_size(n_seqs, hq, hkv, max_ctx, hd)
    if scratch is None:
        scratch = torch.empty(max(need, 1), dtype=torch.uint8, device=q.device)
    n_arena_blocks = k_arena.numel() // (16 * hkv * hd * n_layer)
    _lib.check(_lib.load().dcg_paged_attn_decode(
        _ptr(q), _ptr(k_arena), _ptr(v_arena), n_arena_blocks, n_layer, layer, _ptr(block_tables),
        block_tables.shape[1], _ptr(ctx_lens), n_seqs, hq, hkv, hd, max_ctx, scale, _ptr(out),
        _ptr(scratch), scratch.numel(), _stream()), "dcg_paged_attn_decode")
    return out


def paged_attn_prefill(q: torch.Tensor, k_arena: torch.Tensor, v_arena: torch.Tensor, n_layer: int,
                       layer: int, block_tables: torch.Tensor, seq_starts: torch.Tensor, ctx_lens: torch.Tensor,
                       hkv: int, max_seq_tokens: int, max_ctx: int, scale: float | None = None,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of several new tokens per sequence over the paged fp16 KV arena.

    q [n_tok, hq, 128] f32, sequence s's tokens are rows seq_starts[s] .. seq_starts[s+1]-1
    (seq_starts [n_seqs + 1] int32); its i-th new token sits at position ctx_lens[s] - n_s + i
    (K/V already appended) and attends to keys 0 .. that position."""
    _check_cuda(q, "q", torch.float32)
    for t, nm in ((k_arena, "k_arena"), (v_arena, "v_arena")):
        _check_cuda(t, nm, torch.float16)
    for t, nm in ((block_tables, "block_tables"), (seq_starts, "seq_starts"), (ctx_lens, "ctx_lens")):
        _check_cuda(t, nm, torch.int32)
    n_tok, hq, hd = q.shape
    n_seqs = seq_starts.numel() - 1
    if scale is None:
        scale = 1.0 / float(hd) ** 0.5
    if out is None:
        out = torch.empty_like(q)
    n_arena_blocks = k_arena.numel() // (16 * hkv * hd * n_layer)
    _lib.check(_lib.load().dcg_paged_attn_prefill(
        _ptr(q), _ptr(k_arena), _ptr(v_arena), n_arena_blocks, n_layer, layer, _ptr(block_tables),
        block_tables.shape[1], _ptr(seq_starts), _ptr(ctx_lens), n_seqs, max_seq_tokens, hq, hkv, hd, max_ctx,
        scale, _ptr(out), _stream()), "dcg_paged_attn_prefill")
    return out


def kv_append(k: torch.Tensor, v: torch.Tensor, k_arena: torch.Tensor, v_arena: torch.Tensor,
              n_layer: int, layer: int, block_tables: torch.Tensor, seq_ids: torch.Tensor,
              positions: torch.Tensor) -> None:
    """Write n_tok tokens' K/V ([n_tok, hkv, hd] f32) into their fp16 slots (in place)."""
    for t, nm in ((k, "k"), (v, "v")):
        _check_cuda(t, nm, torch.float32)
    n_tok, hkv, hd = k.shape
    _lib.check(_lib.load().dcg_kv_append(
        _ptr(k), _ptr(v), _ptr(k_arena), _ptr(v_arena), n_layer, layer, _ptr(block_tables),
        block_tables.shape[1], _ptr(seq_ids), _ptr(positions), n_tok, hkv, hd, _stream()),
        "dcg_kv_append")


def _check_all(dev: int, *named):
    """(tensor, name, dtype) triples: contiguous tensors of that type on CUDA device `dev` (its index).
    These checks are most of a small call's time: one pass, no tensor touched twice."""
    for t, name, dtype in named:
        if t.dtype is not dtype or t.get_device() != dev or dev < 0 or not t.is_contiguous():
            _check_cuda(t, name, dtype)
            raise ValueError(f"{name} is on {t.device}, expected cuda:{dev}")


def _call(dev: int, fn: str, *args):
    """Call a device entry point on `dev` and its current stream (whatever device is current)."""
    stream = torch._C._cuda_getCurrentRawStream(dev)   # a Stream object costs more than a launch
    if dev == torch._C._cuda_getDevice():
        rc = getattr(_lib.load(), fn)(*args, stream)
    else:
        with torch.cuda.device(dev):
            rc = getattr(_lib.load(), fn)(*args, stream)
    if rc:
        _lib.check(rc, fn)


def _arena_shape(k_arena: torch.Tensor, v_arena: torch.Tensor, n_layer: int):
    """(blocks, hkv, head_dim) of a pair of arenas [blocks * n_layer, 16, hkv, head_dim]."""
    shape = k_arena.shape
    if len(shape) != 4 or shape[1] != 16 or n_layer < 1 or shape[0] % n_layer:
        raise ValueError(f"arenas must be [blocks * n_layer, 16, hkv, head_dim], got {tuple(shape)}")
    if v_arena.shape != shape:
        raise ValueError("k_arena and v_arena differ in shape")
    return shape[0] // n_layer, shape[2], shape[3]


def tree_masks(parents) -> torch.Tensor:
    """Mask rows of a drafted tree: parents[i] < i is the parent of token i (-1: the history), and
    every token sees its ancestors and itself.  int64 [n, ceil(n / 64)] (CPU), for paged_attn_tree."""
    n = len(parents)
    words = max(1, (n + 63) // 64)
    bits = []
    for i, p in enumerate(parents):
        if not -1 <= p < i:
            raise ValueError(f"parents[{i}] = {p}: a token's parent comes before it (or is -1)")
        bits.append((bits[p] if p >= 0 else 0) | (1 << i))
    rows = np.array([[(b >> (64 * w)) & 0xFFFFFFFFFFFFFFFF for w in range(words)] for b in bits], dtype=np.uint64)
    return torch.from_numpy(rows.reshape(n, words).view(np.int64))


def paged_attn_tree_scratch_size(n_seqs: int, hq: int, hkv: int, max_seq_tokens: int, max_ctx: int,
                                 head_dim: int = 128) -> int:
    return int(_lib.load().dcg_paged_attn_tree_scratch_size(n_seqs, hq, hkv, head_dim, max_seq_tokens, max_ctx))


def paged_attn_tree(q: torch.Tensor, k_arena: torch.Tensor, v_arena: torch.Tensor, n_layer: int, layer: int,
                    block_tables: torch.Tensor, seq_starts: torch.Tensor, ctx_lens: torch.Tensor,
                    tree_mask: torch.Tensor, hkv: int, max_seq_tokens: int, max_ctx: int,
                    scale: float | None = None, out: torch.Tensor | None = None,
                    scratch: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of drafted token trees over the paged fp16 KV arena.

    q [n_tok, hq, 128] f32, sequence s's drafted tokens are rows seq_starts[s] .. seq_starts[s+1]-1;
    token t's K/V sit in slot ctx_lens[s] - n_s + t (already appended).  Row i sees the history and
    drafted token t of its sequence where bit t % 64 of tree_mask[i, t // 64] (int64) is set; a row
    that sees nothing is zeros (see dcg_paged_attn_tree)."""
    dev = q.get_device()
    _check_all(dev, (q, "q", torch.float32), (k_arena, "k_arena", torch.float16), (v_arena, "v_arena", torch.float16),
               (block_tables, "block_tables", torch.int32), (seq_starts, "seq_starts", torch.int32),
               (ctx_lens, "ctx_lens", torch.int32), (tree_mask, "tree_mask", torch.int64))
    shape, tables, words = q.shape, block_tables.shape, tree_mask.shape
    if len(shape) != 3 or len(tables) != 2 or len(words) != 2:
        raise ValueError("q must be [n_tok, hq, head_dim], block_tables and tree_mask two-dimensional")
    n_tok, hq, hd = shape
    n_seqs, mbs = tables
    if seq_starts.numel() != n_seqs + 1 or ctx_lens.numel() != n_seqs:
        raise ValueError("seq_starts needs one entry more than block_tables has rows, ctx_lens as many")
    if words[0] != n_tok:
        raise ValueError("tree_mask needs a row for each row of q")
    for arena in (k_arena.shape, v_arena.shape):   # another form than dcg_kv_fork's is taken by its size
        if len(arena) == 4 and arena[1] == 16 and (arena[2] != hkv or arena[3] != hd):
            raise ValueError(f"arenas of {arena[2]} kv heads x {arena[3]}, called with {hkv} x {hd}")
    per_block = 16 * hkv * hd * n_layer
    elements = k_arena.numel()
    if per_block <= 0 or elements % per_block or v_arena.numel() != elements:
        raise ValueError("arenas are not whole blocks of n_layer x 16 x hkv x head_dim")
    if scale is None:
        scale = 1.0 / float(hd) ** 0.5
    if out is None:
        out = torch.empty_like(q)
    else:
        _check_all(dev, (out, "out", torch.float32))
        if out.shape != shape:
            raise ValueError("out must have q's shape")
    if scratch is None:
        scratch = torch.empty(max(1, paged_attn_tree_scratch_size(n_seqs, hq, hkv, max_seq_tokens, max_ctx, hd)), dtype=torch.uint8, device=f"cuda:{dev}")
    else:
        _check_all(dev, (scratch, "scratch", torch.uint8))
    _call(dev, "dcg_paged_attn_tree", q.data_ptr(), k_arena.data_ptr(), v_arena.data_ptr(),
          elements // per_block, n_layer, layer, block_tables.data_ptr(), mbs,
          seq_starts.data_ptr(), ctx_lens.data_ptr(), tree_mask.data_ptr(), words[1], n_tok, n_seqs,
          max_seq_tokens, hq, hkv, hd, max_ctx, scale, out.data_ptr(), scratch.data_ptr(), scratch.numel())
    return out


def kv_fork_scratch_size(n_seqs: int, max_blocks_per_seq: int, n_arena_blocks: int) -> int:
    return int(_lib.load().dcg_kv_fork_scratch_size(n_seqs, max_blocks_per_seq, n_arena_blocks))


def kv_fork(k_arena: torch.Tensor, v_arena: torch.Tensor, n_layer: int, block_tables: torch.Tensor,
            ctx_lens: torch.Tensor, n_pages: torch.Tensor, ref_counts: torch.Tensor, parents: torch.Tensor,
            reserve: torch.Tensor | None = None, fill_page: int = 0, status: torch.Tensor | None = None,
            scratch: torch.Tensor | None = None) -> torch.Tensor:
    """Row i of the table becomes a child of row parents[i] (-1: empty), in place: it shares the
    parent's blocks, gets a copy of a partly filled last block that others hold too, and the blocks
    that ctx_len + reserve[i] tokens need; blocks nobody holds any more are free.  All of
    block_tables, ctx_lens, n_pages, ref_counts are int32 and updated in place; the arenas are
    [blocks * n_layer, 16, hkv, head_dim] fp16.  Returns status (int32): 0, or the number of blocks
    that were missing, or -1 for bad input; unless 0 nothing was changed (see dcg_kv_fork)."""
    dev = k_arena.get_device()
    i32 = torch.int32
    _check_all(dev, (k_arena, "k_arena", torch.float16), (v_arena, "v_arena", torch.float16),
               (block_tables, "block_tables", i32), (ctx_lens, "ctx_lens", i32), (n_pages, "n_pages", i32),
               (ref_counts, "ref_counts", i32), (parents, "parents", i32))
    blocks, hkv, hd = _arena_shape(k_arena, v_arena, n_layer)
    tables = block_tables.shape
    if len(tables) != 2:
        raise ValueError("block_tables must be two-dimensional")
    n, mbs = tables
    if ctx_lens.numel() != n or n_pages.numel() != n or parents.numel() != n:
        raise ValueError("ctx_lens, n_pages and parents need an entry for each row of block_tables")
    if ref_counts.numel() != blocks:
        raise ValueError(f"ref_counts has {ref_counts.numel()} entries, the arenas hold {blocks} blocks")
    if reserve is not None:
        _check_all(dev, (reserve, "reserve", i32))
        if reserve.numel() != n:
            raise ValueError("reserve needs an entry for each row of block_tables")
    if status is None:
        status = torch.empty((), dtype=i32, device=f"cuda:{dev}")
    else:
        _check_all(dev, (status, "status", i32))
        if status.numel() < 1:
            raise ValueError("status must hold one int32")
    if scratch is None:
        scratch = torch.empty(max(1, kv_fork_scratch_size(n, mbs, blocks)), dtype=torch.uint8, device=f"cuda:{dev}")
    else:
        _check_all(dev, (scratch, "scratch", torch.uint8))
    _call(dev, "dcg_kv_fork", k_arena.data_ptr(), v_arena.data_ptr(), blocks, n_layer, hkv, hd,
          block_tables.data_ptr(), mbs, ctx_lens.data_ptr(), n_pages.data_ptr(), ref_counts.data_ptr(),
          parents.data_ptr(), reserve.data_ptr() if reserve is not None else None, n, fill_page,
          status.data_ptr(), scratch.data_ptr(), scratch.numel())
    return status


def kv_compact(k_arena: torch.Tensor, v_arena: torch.Tensor, n_layer: int, block_tables: torch.Tensor,
               base_lens: torch.Tensor, path: torch.Tensor, path_lens: torch.Tensor, ctx_lens: torch.Tensor) -> None:
    """Move accepted drafted tokens together: slot base_lens[s] + path[s, j] of sequence s goes to
    slot base_lens[s] + j for j < path_lens[s], in every layer, and ctx_lens[s] becomes
    base_lens[s] + path_lens[s] (in place; int32; see dcg_kv_compact)."""
    dev = k_arena.get_device()
    i32 = torch.int32
    _check_all(dev, (k_arena, "k_arena", torch.float16), (v_arena, "v_arena", torch.float16),
               (block_tables, "block_tables", i32), (base_lens, "base_lens", i32), (path, "path", i32),
               (path_lens, "path_lens", i32), (ctx_lens, "ctx_lens", i32))
    blocks, hkv, hd = _arena_shape(k_arena, v_arena, n_layer)
    tables, paths = block_tables.shape, path.shape
    if len(tables) != 2 or len(paths) != 2:
        raise ValueError("block_tables and path must be two-dimensional")
    n = tables[0]
    if base_lens.numel() != n or paths[0] != n or path_lens.numel() != n or ctx_lens.numel() != n:
        raise ValueError("base_lens, path, path_lens and ctx_lens need an entry for each row of block_tables")
    _call(dev, "dcg_kv_compact", k_arena.data_ptr(), v_arena.data_ptr(), blocks, n_layer, hkv, hd,
          block_tables.data_ptr(), tables[1], base_lens.data_ptr(), path.data_ptr(), paths[1],
          path_lens.data_ptr(), n, ctx_lens.data_ptr())


def beam_select_scratch_size(n_groups: int, n_beams: int, vocab: int, k: int) -> int:
    return int(_lib.load().dcg_beam_select_scratch_size(n_groups, n_beams, vocab, k))


def beam_select(logits: torch.Tensor, scores: torch.Tensor, n_beams: int, k: int,
                finished: torch.Tensor | None = None, eos: int = -1, out: tuple | None = None,
                scratch: torch.Tensor | None = None):
    """The k best continuations of each group of n_beams beams.

    logits [n_groups * n_beams, vocab] f32 (rows may be strided), scores [n_groups * n_beams] f32;
    candidates score scores[row] + log_softmax(logits[row])[token].  Returns (scores [n_groups, k]
    f32, rows int32, tokens int32), best first; rows index `logits` (the parents for kv_fork).
    finished (uint8): a finished row offers itself alone, as token eos (see dcg_beam_select)."""
    dev = logits.get_device()
    if dev < 0 or logits.dtype != torch.float32 or logits.dim() != 2 or logits.stride(1) != 1:
        raise ValueError("logits must be a two-dimensional CUDA tensor of float32 with contiguous rows")
    rows, vocab = logits.shape
    if n_beams < 1 or rows % n_beams:
        raise ValueError(f"{rows} rows of logits are not whole groups of {n_beams} beams")
    groups = rows // n_beams
    _check_all(dev, (scores, "scores", torch.float32))
    if scores.numel() != rows:
        raise ValueError("scores needs an entry for each row of logits")
    if finished is not None:
        _check_all(dev, (finished, "finished", torch.uint8))
        if finished.numel() != rows:
            raise ValueError("finished needs an entry for each row of logits")
    if out is None:
        out = (torch.empty((groups, k), dtype=torch.float32, device=f"cuda:{dev}"),
               torch.empty((groups, k), dtype=torch.int32, device=f"cuda:{dev}"),
               torch.empty((groups, k), dtype=torch.int32, device=f"cuda:{dev}"))
    else:
        _check_all(dev, (out[0], "out scores", torch.float32), (out[1], "out rows", torch.int32),
                   (out[2], "out tokens", torch.int32))
        if any(t.numel() != groups * k for t in out):
            raise ValueError("out tensors must hold n_groups * k values")
    if scratch is None:
        scratch = torch.empty(max(1, beam_select_scratch_size(groups, n_beams, vocab, k)), dtype=torch.uint8, device=f"cuda:{dev}")
    else:
        _check_all(dev, (scratch, "scratch", torch.uint8))
    _call(dev, "dcg_beam_select", logits.data_ptr(), logits.stride(0) if rows > 1 else max(vocab, logits.stride(0)),
          groups, n_beams, vocab, scores.data_ptr(), finished.data_ptr() if finished is not None else None, eos, k,
          out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), scratch.data_ptr(), scratch.numel())
    return out


def add_rmsnorm_quantize(x: torch.Tensor, weight: torch.Tensor, eps: float, act_type: int,
                         act: torch.Tensor, delta: torch.Tensor | None = None) -> torch.Tensor:
    """x += delta (in place, optional); act = quantize(rmsnorm(x) * weight)."""
    m, k = x.shape
    _lib.check(_lib.load().dcg_add_rmsnorm_quantize(
        _ptr(x), _ptr(delta) if delta is not None else None, _ptr(weight), eps, m, k, act_type,
        _ptr(act), _stream()), "dcg_add_rmsnorm_quantize")
    return act


def swiglu_quantize(gate: torch.Tensor, up: torch.Tensor, ld: int, m: int, ffn: int, act_type: int,
                    act: torch.Tensor) -> torch.Tensor:
    """act = quantize(silu(gate) * up) over rows of `ffn` values with row stride `ld`."""
    _lib.check(_lib.load().dcg_swiglu_quantize(_ptr(gate), _ptr(up), ld, m, ffn, act_type, _ptr(act),
                                               _stream()), "dcg_swiglu_quantize")
    return act


def qk_norm_rope_kv_append(q, ldq, k, ldk, v, ldv, n_seqs, hq, hkv, q_norm_w, k_norm_w, eps, theta,
                           positions, q_out, k_arena, v_arena, n_layer, layer, block_tables):
    """Per-head RMSNorm + NeoX RoPE of q and k; q -> q_out, k/v -> fp16 paged slots."""
    _lib.check(_lib.load().dcg_qk_norm_rope_kv_append(
        _ptr(q), ldq, _ptr(k), ldk, _ptr(v), ldv, n_seqs, hq, hkv, 128,
        _ptr(q_norm_w) if q_norm_w is not None else None,
        _ptr(k_norm_w) if k_norm_w is not None else None,
        eps, theta, _ptr(positions), _ptr(q_out), _ptr(k_arena), _ptr(v_arena), n_layer, layer,
        _ptr(block_tables), block_tables.shape[1], _stream()), "dcg_qk_norm_rope_kv_append")


def qk_norm_rope_kv_append_tokens(q, ldq, k, ldk, v, ldv, n_tok, hq, hkv, q_norm_w, k_norm_w, eps, theta,
                                  seq_ids, positions, q_out, k_arena, v_arena, n_layer, layer, block_tables):
    """qk_norm_rope_kv_append for token rows of any sequences (row i: sequence seq_ids[i])."""
    _lib.check(_lib.load().dcg_qk_norm_rope_kv_append_tokens(
        _ptr(q), ldq, _ptr(k), ldk, _ptr(v), ldv, n_tok, hq, hkv, 128,
        _ptr(q_norm_w) if q_norm_w is not None else None,
        _ptr(k_norm_w) if k_norm_w is not None else None,
        eps, theta, _ptr(seq_ids), _ptr(positions), _ptr(q_out), _ptr(k_arena), _ptr(v_arena), n_layer, layer,
        _ptr(block_tables), block_tables.shape[1], _stream()), "dcg_qk_norm_rope_kv_append_tokens")


def qk_norm_rope_kv_append_tree(q, ldq, k, ldk, v, ldv, n_tok, hq, hkv, q_norm_w, k_norm_w, eps, theta,
                                seq_ids, positions, slots, q_out, k_arena, v_arena, n_layer, layer, block_tables):
    """qk_norm_rope_kv_append_tokens with the cache slot of each row apart from its position."""
    _lib.check(_lib.load().dcg_qk_norm_rope_kv_append_tree(
        _ptr(q), ldq, _ptr(k), ldk, _ptr(v), ldv, n_tok, hq, hkv, 128,
        _ptr(q_norm_w) if q_norm_w is not None else None,
        _ptr(k_norm_w) if k_norm_w is not None else None,
        eps, theta, _ptr(seq_ids), _ptr(positions), _ptr(slots), _ptr(q_out), _ptr(k_arena), _ptr(v_arena), n_layer,
        layer, _ptr(block_tables), block_tables.shape[1], _stream()), "dcg_qk_norm_rope_kv_append_tree")


class HostContext:
    """The synchronous host boundary: weights registered once by host pointer, per-call host
    activations in and host results out (dcg_ctx_*)."""

    def __init__(self, device: int = 0):
        self._L = _lib.load()
        h = ctypes.c_void_p()
        _lib.check(self._L.dcg_ctx_create(device, ctypes.byref(h)), "dcg_ctx_create")
        self.h = h
        self._keep = {}
        self._mm = self._L.dcg_ctx_mul_mat

    def register(self, rows: np.ndarray, qtype: int, k: int):
        rows = np.ascontiguousarray(rows, dtype=np.uint8)
        n = rows.shape[0]
        w = ctypes.c_void_p()
        _lib.check(self._L.dcg_ctx_weight_register(self.h, qtype, rows.ctypes.data, rows.strides[0],
                                                   n, k, ctypes.byref(w)),
                   "dcg_ctx_weight_register")
        self._keep[w.value] = (rows, n, k)
        return w

    def mul_mat(self, w, x: np.ndarray) -> np.ndarray:
        rows, n, k = self._keep[w.value]
        if not (x.dtype == np.float32 and x.flags.c_contiguous):
            x = np.ascontiguousarray(x, dtype=np.float32)
        m = x.size // k
        if m * k != x.size:
            raise ValueError(f"x has {x.size} elements, not a multiple of k={k}")
        y = np.empty((m, n), dtype=np.float32)
        rc = self._mm(self.h, w, x.ctypes.data, m, y.ctypes.data)
        if rc:
            _lib.check(rc, "dcg_ctx_mul_mat")
        return y

    def close(self):
        if self.h:
            self._L.dcg_ctx_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
