"""Further refusals and host logic of the branching operators, decided without a GPU."""
import types

import pytest
import torch

import branch_ref as R
from densecore_b200 import _lib, batching, ops
from test_branch_cpu import EINVAL, P, beam, compact, fork, tree


# base_lens, path_lens 8 bytes, path and block_tables 32 at P
@pytest.mark.parametrize("kw", [
    dict(base=4 * P, path=4 * P, bt=4 * P, ctx=P), dict(base=4 * P, path=4 * P, bt=4 * P, ctx=P - 4),
    dict(base=4 * P, plens=4 * P, bt=4 * P, ctx=P + 28), dict(base=4 * P, plens=4 * P, path=4 * P, ctx=P + 28)])
def test_compact_refuses_lengths_that_overlap_what_it_reads(kw):
    assert compact(**kw) == EINVAL
    assert b"overlap" in _lib.load().dcg_last_error()


APART = dict(bt=2 * P, lens=3 * P, held=4 * P, refs=5 * P, parents=6 * P, status=7 * P)   # of fork's arrays: 32 bytes at most


@pytest.mark.parametrize("kw", [dict(parents=2 * P + 24), dict(parents=3 * P), dict(parents=4 * P - 4), dict(parents=5 * P + 28),
                                dict(parents=7 * P - 4), dict(reserve=5 * P + 28)])
def test_fork_refuses_parents_that_it_would_write(kw):
    assert fork(**{**APART, **kw}) == EINVAL
    assert b"overlap" in _lib.load().dcg_last_error()


# two groups of three beams, k 4: 24 bytes of scores, 6 of flags, 32 of each result
@pytest.mark.parametrize("kw", [dict(s=2 * P), dict(s=2 * P + 20), dict(s=2 * P - 28), dict(r=2 * P), dict(t=2 * P + 20), dict(k=3, s=2 * P + 12),
                                dict(s=3 * P), dict(r=3 * P + 4), dict(t=3 * P - 28)])
def test_beam_refuses_results_over_what_it_reads(kw):
    apart = dict(scores=2 * P, finished=3 * P, s=4 * P, r=5 * P, t=6 * P)
    assert beam(**{**apart, **kw}) == EINVAL
    assert b"overlap" in _lib.load().dcg_last_error()


@pytest.mark.parametrize("off", [16, -16, 4 * 16 * 512 - 16])      # 4 tokens of 16 heads
def test_tree_refuses_an_output_across_q(off):
    assert tree(q=1 << 20, out=(1 << 20) + off) == EINVAL
    assert b"overlap" in _lib.load().dcg_last_error()


# ------------------------------------------------------------------------- host logic of the loops
VOCAB = 50


def follows(history):
    """The next token of a text: the fakes' model."""
    return (sum((i + 3) * (t + 1) for i, t in enumerate(history[-5:])) + len(history)) % VOCAB


class FakeDecoder:
    """A decoder on the CPU whose cache holds tokens: every prediction is read back through the block
    table, slot by slot, so a block that went to two rows or was given away shows."""

    def __init__(self, batch, max_ctx, n_blocks=None):
        self.batch, self.max_ctx, self.device = batch, max_ctx, "cpu"
        self.cfg = types.SimpleNamespace(n_layer=1, vocab=VOCAB)
        self.blocks_per_seq = -(-max_ctx // 16)
        self.n_blocks = n_blocks or batch * self.blocks_per_seq + 1
        self.block_tables = torch.arange(batch * self.blocks_per_seq, dtype=torch.int32).view(batch, -1) % self.n_blocks
        self.k_arena = torch.zeros((self.n_blocks, 16), dtype=torch.long)
        self.v_arena = self.k_arena

    def _put(self, s, at, token):
        self.k_arena[self.block_tables[s, at // 16], at % 16] = token

    def _history(self, s, n):
        return [int(self.k_arena[self.block_tables[s, j // 16], j % 16]) for j in range(n)]

    def prefill(self, seqs, prompts):
        for s, p in zip(seqs, prompts):
            for j, t in enumerate(p):
                self._put(s, j, t)
        return torch.tensor([follows(self._history(s, len(p))) for s, p in zip(seqs, prompts)]), None

    def verify_tree(self, seqs, trees, start):
        for s, (tokens, _), base in zip(seqs, trees, start):
            assert base + len(tokens) <= self.max_ctx
            for j, t in enumerate(tokens):
                self._put(s, base + j, t)
        out = []
        for s, (tokens, parents), base in zip(seqs, trees, start):
            text = self._history(s, base + len(tokens))
            for j in range(len(tokens)):
                branch, i = [], j
                while i >= 0:
                    branch.append(text[base + i])
                    i = parents[i]
                out.append(follows(text[:base] + branch[::-1]))
        return torch.tensor(out), None


def fake_fork(k, v, n_layer, tables, lens, held, refs, parents, reserve=None, fill_page=0, status=None, scratch=None):
    want = R.fork(tables.tolist(), refs.tolist(), lens.tolist(), held.tolist(), parents.tolist(),
                  reserve.tolist() if reserve is not None else [0] * len(lens), fill_page)
    for t, w in zip((tables, refs, lens, held), want):
        t.copy_(torch.tensor(w, dtype=torch.int32))
    for src, dst, slots in want[4]:
        k[dst, :slots] = k[src, :slots].clone()
    status.fill_(want[5])


def fake_compact(k, v, n_layer, tables, base, path, path_lens, lens):
    for s, n in enumerate(path_lens.tolist()):
        for j in range(n):
            at, to = int(base[s] + path[s, j]), int(base[s]) + j
            k[tables[s, to // 16], to % 16] = k[tables[s, at // 16], at % 16].clone()
        lens[s] = base[s] + n


@pytest.fixture
def on_cpu(monkeypatch):
    monkeypatch.setattr(ops, "kv_fork", fake_fork)
    monkeypatch.setattr(ops, "kv_compact", fake_compact)


def greedy(prompt, n, eos=None):
    out = []
    while len(out) < n and (not out or out[-1] != eos):
        out.append(follows(prompt + out))
    return out


def test_pool_tells_bad_input_from_too_few_blocks(on_cpu):
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    pool = batching.PagePool(FakeDecoder(2, 64, 4))
    pool.check()
    pool.fork(i32(2, 0))
    with pytest.raises(ValueError, match="out of range"):
        pool.check()
    pool = batching.PagePool(FakeDecoder(2, 64, 4))
    pool.fork(reserve=i32(40, 40))
    pool.fork(i32(5, 0))                     # the first thing that went wrong is what is told
    with pytest.raises(MemoryError, match="3 blocks"):
        pool.check()


def test_pool_gives_the_table_back(on_cpu):
    dec = FakeDecoder(2, 64)
    before = dec.block_tables.clone()
    prompts = [[1, 2, 3] * 7, [4] * 18]
    assert batching.TreeSpeculator(dec).generate(prompts, 20) == [greedy(p, 20) for p in prompts]
    assert torch.equal(dec.block_tables, before)
    with batching.PagePool(dec) as pool:
        pool.fork(reserve=torch.full((2,), 17, dtype=torch.int32))
        assert not torch.equal(dec.block_tables, before)
    assert torch.equal(dec.block_tables, before)

    def broken(history):
        raise RuntimeError("no draft")
    with pytest.raises(RuntimeError):
        batching.TreeSpeculator(dec, broken).generate(prompts, 20)
    assert torch.equal(dec.block_tables, before)
