"""Further refusals and host logic of the branching operators, decided without a GPU."""
import random
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


def wild(history):
    """Forty guesses, nearly all of them wrong."""
    rng = random.Random(len(history))
    return [rng.randrange(VOCAB) for _ in range(40)], [rng.randrange(-1, i) if i else -1 for i in range(40)]


class Watched(batching.PagePool):
    """A pool that looks at its books after every fork: what a row holds is what it needs, every block's count is
    the number of rows that hold it."""

    forks = 0

    def fork(self, parents=None, reserve=None):
        super().fork(parents, reserve)
        type(self).forks += 1
        room = self.lens + (reserve if reserve is not None else 0)
        assert torch.equal(self.pages, torch.where(self.lens + (parents if parents is not None else 0) < 0, 0, -(-room // 16)))
        held = [0] * self.dec.n_blocks
        held[0] = 1
        for row, n in zip(self.tables.tolist(), self.pages.tolist()):
            for b in row[:n]:
                held[b] += 1
        assert self.refs.tolist() == held and max(held) == 1


@pytest.mark.parametrize("draft", [wild, batching.ngram_draft])
def test_speculator_in_a_tight_arena(on_cpu, monkeypatch, draft):
    """Drafts never take a block that the text needs: an arena that holds the finished texts is enough."""
    monkeypatch.setattr(batching, "PagePool", Watched)
    prompts = [[1] * 30, [2] * 30, [3] * 7]
    need = sum(-(-(len(p) + 34) // 16) for p in prompts)      # the last token is not in the cache
    dec = FakeDecoder(4, 96, need + 1)
    assert batching.TreeSpeculator(dec, draft).generate(prompts, 35) == [greedy(p, 35) for p in prompts]
    # one block short of that: nothing is lost if a text ends early enough, and another waits for it
    eos = greedy(prompts[0], 35)[3]
    want = [greedy(p, 35, eos) for p in prompts]
    assert len(want[0]) == 4 and batching.TreeSpeculator(FakeDecoder(4, 96, need), draft).generate(prompts, 35, eos) == want
    small = FakeDecoder(1, 96, 4)
    before = small.block_tables.clone()
    with pytest.raises(MemoryError):
        batching.TreeSpeculator(small, draft).generate([[1] * 30], 35)
    assert torch.equal(small.block_tables, before) and Watched.forks


def test_speculator_gives_every_block_back(on_cpu, monkeypatch):
    """Rejected drafts, rows that end at different times and at eos: no block stays held."""
    pools = []

    class Kept(Watched):
        def close(self):
            self.fork(torch.full((self.dec.batch,), -1, dtype=torch.int32))
            pools.append(self.refs.tolist())
            super().close()
    monkeypatch.setattr(batching, "PagePool", Kept)
    prompts = [[7, 8, 9], [5] * 40, [6] * 16]
    eos = greedy(prompts[2], 30)[11]
    for e in (None, eos):
        dec = FakeDecoder(4, 96)
        assert batching.TreeSpeculator(dec, wild).generate(prompts, 30, e) == [greedy(p, 30, e) for p in prompts]
    assert pools == [[1] + [0] * (dec.n_blocks - 1)] * 2


def test_speculator_rows_wait_for_blocks(on_cpu, monkeypatch):
    """Two texts that do not fit side by side: the second goes on when the first has ended."""
    monkeypatch.setattr(batching, "PagePool", Watched)
    eos = greedy([1] * 15, 17)[16]
    long = next([t] * 32 for t in range(VOCAB) if eos not in greedy([t] * 32, 40))
    prompts = [[1] * 15, long]
    want = [greedy(p, 40, eos) for p in prompts]
    assert len(want[0]) == 17 and len(want[1]) == 40
    # idle, two blocks each, one more for the second
    for n_blocks in (5, 6):
        assert batching.TreeSpeculator(FakeDecoder(2, 96, n_blocks + 1), wild).generate(prompts, 40, eos) == want


@pytest.mark.parametrize("seqs,trees,start,word", [
    ([0, 0], [([1], [-1])] * 2, [5, 5], "different rows"), (torch.tensor([2, 2]), [([1], [-1])] * 2, [5, 5], "different rows"),
    ([0, 3], [([1], [-1])] * 2, [5, 5], "different rows"),
    ([-1], [([1], [-1])], [5], "different rows"), ([1], [([1], [-1])], [-1], "start"), ([1], [([1, 50], [-1, 0])], [5], "tokens"),
    ([1], [([1, -1], [-1, 0])], [5], "tokens"), ([1], [([1, 2], [-1])], [5], "parent"), ([1], [([1], [-1])], [5, 6], "length")])
def test_verify_tree_refuses(seqs, trees, start, word):
    """On the host, before anything is looked up on the device."""
    from densecore_b200.decoder import Decoder
    dec = Decoder.__new__(Decoder)
    dec.batch, dec.tp_size, dec.cfg = 3, 1, types.SimpleNamespace(vocab=VOCAB)
    with pytest.raises(ValueError, match=word):
        dec.verify_tree(seqs, trees, start)


@pytest.mark.parametrize("bad", [-1, VOCAB])
def test_loops_refuse_tokens_beyond_the_vocabulary(on_cpu, bad):
    dec = FakeDecoder(2, 64)
    with pytest.raises(ValueError, match="tokens"):
        batching.TreeSpeculator(dec).generate([[1, 2], [3, bad]], 5)
    with pytest.raises(ValueError, match="tokens"):
        batching.BeamSearcher(dec, 1).search([[1, 2], [bad]], 5)
