"""Refusals of the branching operators (tree attention, page forking, slot compaction, beam
selection) and the host helper for masks: everything that is decided without a GPU."""
import numpy as np
import pytest
import torch

from densecore_b200 import _lib, ops

EINVAL, ESCRATCH = -1, -4
P = 4096   # a non-null, aligned stand-in for a device pointer: no refused call reads it


def tree(**kw):
    a = dict(q=P, k=P, v=P, blocks=8, n_layer=2, layer=1, bt=P, mbs=4, starts=P, ctx=P, mask=P, words=1, n_tok=4,
             n_seqs=1, max_tok=4, hq=16, hkv=8, hd=128, max_ctx=64, scale=0.1, out=P, scratch=P, nbytes=1 << 40)
    a.update(kw)
    return _lib.load().dcg_paged_attn_tree(*a.values(), None)


@pytest.mark.parametrize("kw,word", [
    (dict(q=None), b"null"), (dict(mask=None), b"null"), (dict(hd=64), b"head_dim"), (dict(hq=12), b"multiple"),
    (dict(hkv=0), b"multiple"), (dict(layer=2), b"layer"), (dict(blocks=0), b"n_arena_blocks"),
    (dict(blocks=1 << 28), b"n_arena_blocks"), (dict(max_ctx=65), b"block table"), (dict(max_tok=65), b"words"),
    (dict(words=0), b"words"), (dict(q=P + 4), b"aligned"), (dict(mask=P + 4), b"aligned"), (dict(n_seqs=-1), b">= 0"),
    (dict(n_seqs=70000), b"65535"), (dict(mbs=0), b"max_blocks")])
def test_tree_refuses(kw, word):
    assert tree(**kw) == EINVAL
    assert word in _lib.load().dcg_last_error()


@pytest.mark.parametrize("kw", [dict(n_seqs=65535), dict(hq=65535, hkv=1), dict(n_seqs=65534, hq=40000, hkv=40000)])
def test_tree_refuses_what_a_grid_cannot_hold(kw):
    assert tree(**kw) == EINVAL
    assert b"65535" in _lib.load().dcg_last_error()


def test_tree_without_work_is_ok():
    assert tree(n_seqs=0) == 0 and tree(n_tok=0) == 0 and tree(max_tok=0) == 0


def fork(**kw):
    a = dict(k=P, v=P, blocks=8, n_layer=2, hkv=8, hd=128, bt=P, mbs=4, lens=P, held=P, refs=P, parents=P, reserve=None,
             n=2, fill=0, status=P, scratch=P, nbytes=1 << 40)
    a.update(kw)
    return _lib.load().dcg_kv_fork(*a.values(), None)


@pytest.mark.parametrize("kw,word", [
    (dict(status=None), b"null"), (dict(parents=None), b"null"), (dict(n=-1), b"n_seqs"), (dict(n=4097), b"4096"),
    (dict(fill=8), b"fill_block"), (dict(fill=-1), b"fill_block"), (dict(hkv=1, hd=4), b"multiple of 8"),
    (dict(k=P + 8), b"aligned"), (dict(scratch=P + 16), b"aligned"), (dict(mbs=0), b"shape"),
    (dict(blocks=0), b"shape")])
def test_fork_refuses(kw, word):
    assert fork(**kw) == EINVAL
    assert word in _lib.load().dcg_last_error()


def test_fork_scratch():
    assert fork(nbytes=0) == ESCRATCH
    need = _lib.load().dcg_kv_fork_scratch_size
    assert need(0, 4, 8) == 0 and need(2, 4, 8) >= 2 * 8 * 4
    assert need(64, 4096, 10) < need(64, 4096, 100000)


def compact(**kw):
    a = dict(k=P, v=P, blocks=8, n_layer=2, hkv=8, hd=128, bt=P, mbs=4, base=P, path=P, max_path=4, plens=P, n=2,
             ctx=2 * P)
    a.update(kw)
    return _lib.load().dcg_kv_compact(*a.values(), None)


@pytest.mark.parametrize("kw,word", [
    (dict(path=None), b"null"), (dict(max_path=0), b"max_path"), (dict(max_path=1025), b"max_path"),
    (dict(ctx=P), b"overlap"), (dict(ctx=P + 4), b"overlap"), (dict(n=70000), b"65535"), (dict(n=-1), b"n_seqs"),
    (dict(v=P + 2), b"aligned"), (dict(n_layer=0), b"shape")])
def test_compact_refuses(kw, word):
    assert compact(**kw) == EINVAL
    assert word in _lib.load().dcg_last_error()


def beam(**kw):
    a = dict(x=P, ld=100, groups=2, beams=3, vocab=100, scores=P, finished=None, eos=0, k=4, s=P, r=P, t=P, scratch=P,
             nbytes=1 << 40)
    a.update(kw)
    return _lib.load().dcg_beam_select(*a.values(), None)


@pytest.mark.parametrize("kw,word", [
    (dict(k=0), b"1 .. 64"), (dict(k=65), b"1 .. 64"), (dict(vocab=0), b"vocab"), (dict(beams=0), b"n_beams"),
    (dict(ld=99), b"ld"), (dict(x=None), b"null"), (dict(x=P + 2), b"aligned"), (dict(groups=-1), b"n_groups"),
    (dict(vocab=1 << 31, ld=1 << 31), b"vocab"), (dict(scratch=P + 8), b"aligned")])
def test_beam_refuses(kw, word):
    assert beam(**kw) == EINVAL
    assert word in _lib.load().dcg_last_error()


def test_beam_scratch():
    assert beam(nbytes=0) == ESCRATCH and beam(groups=0) == 0
    assert ops.beam_select_scratch_size(2, 3, 100, 65) == 0


def test_wrappers_refuse_cpu_tensors():
    z = torch.zeros
    i = lambda *s: z(s, dtype=torch.int32)  # noqa: E731
    h = z((4, 16, 8, 128), dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attn_tree(z(1, 8, 128), h, h, 1, 0, i(1, 4), i(2), i(1), z((1, 1), dtype=torch.int64), 8, 1, 16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_fork(h, h, 1, i(1, 4), i(1), i(1), i(4), i(1))
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_compact(h, h, 1, i(1, 4), i(1), i(1, 1), i(1), i(1))
    with pytest.raises(ValueError, match="CUDA"):
        ops.beam_select(z(2, 10), z(2), 2, 2)


def test_tree_masks():
    m = ops.tree_masks([-1, 0, 0, 1, -1]).numpy()
    assert m.shape == (5, 1) and m[:, 0].tolist() == [1, 3, 5, 11, 16]
    deep = ops.tree_masks([i - 1 for i in range(130)]).numpy().view(np.uint64)
    assert deep.shape == (130, 3)
    bits = [int(r[0]) | int(r[1]) << 64 | int(r[2]) << 128 for r in deep]
    assert bits == [(1 << (i + 1)) - 1 for i in range(130)]
    assert ops.tree_masks([]).shape == (0, 1)
    for bad in ([0], [-1, 1], [-2], [-1, 2, 0]):
        with pytest.raises(ValueError):
            ops.tree_masks(bad)


# ------------------------------------------------------------------------- host logic of the loops
def test_accept_path():
    from densecore_b200.batching import accept_path
    #        0   1   2   3   4   5
    tok = [10, 11, 12, 13, 14, 13]
    par = [-1, 0, 0, 2, 3, 1]
    assert accept_path(tok, par, [12, 0, 13, 14, 9, 9]) == [0, 2, 3, 4]
    assert accept_path(tok, par, [11, 13, 0, 0, 0, 0]) == [0, 1, 5]
    assert accept_path(tok, par, [99, 0, 0, 0, 0, 0]) == [0]
    assert accept_path([7], [-1], [3]) == [0]
    # the same guess twice: the first one
    assert accept_path([1, 2, 2], [-1, 0, 0], [2, 5, 5]) == [0, 1]


def test_ngram_draft():
    from densecore_b200.batching import ngram_draft
    t, p = ngram_draft([1, 2, 3, 4, 1, 2, 3, 5, 1, 2], n=2, depth=3, width=4)
    # after the latest "1 2": 3 5 1; before that 3 4 1 (the 3 is shared)
    assert t == [3, 5, 1, 4, 1] and p == [-1, 0, 1, 0, 3]
    assert ngram_draft([1, 2, 3], n=2) == ([], [])
    assert ngram_draft([1], n=2) == ([], []) and ngram_draft([], n=2) == ([], [])
    t, p = ngram_draft([5] * 10, n=2, depth=4, width=2)
    assert all(q < i for i, q in enumerate(p)) and set(t) == {5}
    assert ops.tree_masks(p).shape[0] == len(t)


def test_beam_paths():
    from densecore_b200.batching import beam_paths
    inf = float("inf")
    # one group of three beams, three steps; the last beam is dead
    steps = [([0, 0, 0], [5, 6, 7]), ([1, 0, -1], [8, 9, -1]), ([0, 0, -1], [2, 3, -1])]
    assert beam_paths([-1.0, -2.0, -inf], steps, 3, 1, None) == [[(-1.0, [6, 8, 2]), (-2.0, [6, 8, 3])]]
    assert beam_paths([-1.0, -2.0, -inf], steps, 3, 1, 8) == [[(-1.0, [6, 8]), (-2.0, [6, 8])]]


def test_loops_refuse():
    from densecore_b200.batching import BeamSearcher, TreeSpeculator

    class Dec:
        batch, max_ctx, device = 6, 32, "cpu"
    with pytest.raises(ValueError):
        BeamSearcher(Dec(), 4)
    with pytest.raises(ValueError):
        BeamSearcher(Dec(), 0)
    for prompts, new in (([], 3), ([[1]] * 3, 3), ([[]], 3), ([[1] * 30], 3), ([[1]], 0)):
        with pytest.raises(ValueError):
            BeamSearcher(Dec(), 3).search(prompts, new)
    for prompts, new in (([], 3), ([[1]] * 7, 3), ([[]], 3), ([[1] * 30], 3), ([[1]], 0)):
        with pytest.raises(ValueError):
            TreeSpeculator(Dec()).generate(prompts, new)
    with pytest.raises(ValueError):
        TreeSpeculator(Dec(), max_nodes=0)
    with pytest.raises(ValueError):
        TreeSpeculator(Dec(), max_nodes=2000)
