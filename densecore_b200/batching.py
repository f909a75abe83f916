"""Continuous batching around the captured decode step: requests join and leave a fixed set of
slots between graph replays, each with its own KV blocks.  This is the host loop of DenseCore's
worker (core/src/worker.cpp:365-544: admit, build the batch, compute, sample, retire) with the
per-sequence semantics the reference's batched path lacks -- every sequence reads only its own
positions through its own block table, so its tokens do not depend on what else is in the batch.

A newly admitted request's whole prompt is ingested by one prefill pass (Decoder.prefill: every
matmul at M = prompt tokens, multi-token causal attention), batched over the requests admitted in
the same step; its last token's logits give the first generated token.  With prefill=False prompts
are instead fed one token per step through the decode graph.  Sampling is greedy.  Idle slots
point at one reserved block and run a harmless one-token step.

Sequences that branch: BeamSearcher (beam search over groups of decoder rows) and TreeSpeculator
(greedy decoding that scores drafted token trees) keep the blocks on the device, shared between rows
and counted (PagePool).  Each takes the whole decoder's cache while it runs: what the cache held is
gone afterwards, the decoder's block table is as it was.
"""
from __future__ import annotations

import collections
import dataclasses

import torch

from . import ops
from .decoder import KV_BLOCK, Decoder, check_tokens


class BlockAllocator:
    """Free list over the KV arena's physical blocks (kv_cache.cpp's block pool)."""

    def __init__(self, n_blocks: int):
        self.free = collections.deque(range(n_blocks))
        self.n_blocks = n_blocks

    def alloc(self, n: int) -> list[int] | None:
        if n > len(self.free):
            return None
        return [self.free.popleft() for _ in range(n)]

    def release(self, blocks: list[int]):
        if len(set(blocks)) != len(blocks) or any(b < 0 or b >= self.n_blocks for b in blocks):
            raise ValueError("bad block list")
        self.free.extend(blocks)
        if len(self.free) > self.n_blocks:
            raise ValueError("block released twice")


@dataclasses.dataclass
class Request:
    rid: int
    prompt: list[int]
    max_new: int
    eos: int | None = None
    out: list[int] = dataclasses.field(default_factory=list)
    # runtime state
    slot: int = -1
    blocks: list[int] = dataclasses.field(default_factory=list)
    pos: int = 0          # tokens already written to the cache

    @property
    def capacity(self) -> int:
        return len(self.prompt) + self.max_new

    def next_input(self) -> int:
        return self.prompt[self.pos] if self.pos < len(self.prompt) else self.out[-1]

    def done(self) -> bool:
        return len(self.out) >= self.max_new or (self.eos is not None and self.out and self.out[-1] == self.eos)


class ContinuousBatcher:
    """Runs requests through `dec` (its batch size is the slot count)."""

    def __init__(self, dec: Decoder, prefill: bool = True):
        self.dec = dec
        self.use_prefill = prefill
        self.slots: list[Request | None] = [None] * dec.batch
        self.alloc = BlockAllocator(dec.n_blocks)
        self.idle_block = self.alloc.alloc(1)[0]   # where idle slots write their throw-away token
        self.queue: collections.deque[Request] = collections.deque()
        self.finished: list[Request] = []
        self._bt = torch.full((dec.batch, dec.blocks_per_seq), self.idle_block, dtype=torch.int32)
        self._tok = torch.zeros(dec.batch, dtype=torch.long)
        self._ctx = torch.ones(dec.batch, dtype=torch.int32)
        self._next_id = 0

    def submit(self, prompt: list[int], max_new: int, eos: int | None = None) -> Request:
        if not prompt or max_new < 1:
            raise ValueError("need a non-empty prompt and max_new >= 1")
        r = Request(self._next_id, list(prompt), max_new, eos)
        if r.capacity > self.dec.max_ctx:
            raise ValueError(f"request needs {r.capacity} positions, the decoder holds {self.dec.max_ctx}")
        self._next_id += 1
        self.queue.append(r)
        return r

    def _admit(self) -> list[Request]:
        new = []
        for s in range(len(self.slots)):
            if self.slots[s] is not None or not self.queue:
                continue
            r = self.queue[0]
            blocks = self.alloc.alloc((r.capacity + KV_BLOCK - 1) // KV_BLOCK)
            if blocks is None:
                break                       # wait for blocks to be released (FIFO admission)
            self.queue.popleft()
            r.slot, r.blocks = s, blocks
            self.slots[s] = r
            self._bt[s].fill_(self.idle_block)
            self._bt[s, :len(blocks)] = torch.tensor(blocks, dtype=torch.int32)
            new.append(r)
        return new

    def _retire(self, s: int, r: Request):
        self.alloc.release(r.blocks)
        r.blocks, r.slot = [], -1
        self.slots[s] = None
        # the idle slot's throw-away writes must not land in blocks that now belong to others
        self._bt[s].fill_(self.idle_block)
        self.finished.append(r)

    def step(self) -> bool:
        """Admit waiting requests (prefilling their prompts), run one decode step for every slot,
        retire finished requests.  Returns False when there is nothing left to do."""
        new = self._admit()
        dec = self.dec
        dec.block_tables.copy_(self._bt, non_blocking=False)
        if new and self.use_prefill:
            nxt, _ = dec.prefill([r.slot for r in new], [r.prompt for r in new])
            for r, t in zip(new, nxt.tolist()):
                r.pos = len(r.prompt)
                r.out.append(int(t))
                if r.done():
                    self._retire(r.slot, r)
        active = [r for r in self.slots if r is not None]
        if not active:
            return bool(self.queue)
        for s, r in enumerate(self.slots):
            if r is None:
                self._tok[s], self._ctx[s] = 0, 1
            else:
                self._tok[s], self._ctx[s] = r.next_input(), r.pos + 1
        dec.tokens.copy_(self._tok)
        dec.ctx_lens.copy_(self._ctx)
        dec.replay()
        nxt = dec.next_tokens.cpu()
        for s, r in enumerate(self.slots):
            if r is None:
                continue
            r.pos += 1
            if r.pos >= len(r.prompt):      # the last prompt token and every generated one predict
                r.out.append(int(nxt[s]))
            if r.done():
                self._retire(s, r)
        return True

    def run(self, max_steps: int = 1 << 30) -> list[Request]:
        n = 0
        while n < max_steps and self.step():
            n += 1
        return self.finished


class PagePool:
    """The decoder's KV blocks as pages shared between rows, kept on the device: the block table, how
    many tokens and blocks each row holds, and how often each block is held.  fork and compact are
    kv_fork and kv_compact on all rows at once; block 0 is the idle block that unused entries point
    at.  Nothing waits for the host except `check`.  The table is the decoder's own; `close` (or the end
    of a with block) puts back what it held before."""

    def __init__(self, dec: Decoder):
        self.dec = dec
        dev, i32 = dec.device, torch.int32
        self.tables = dec.block_tables
        self.lens = torch.zeros(dec.batch, dtype=i32, device=dev)       # tokens in the cache
        self.pages = torch.zeros(dec.batch, dtype=i32, device=dev)
        self.refs = torch.zeros(dec.n_blocks, dtype=i32, device=dev)
        self.refs[0] = 1
        self._before = self.tables.clone()
        self.tables.zero_()
        self.identity = torch.arange(dec.batch, dtype=i32, device=dev)
        self.short = torch.zeros((), dtype=i32, device=dev)             # first status that was not 0
        self._status = torch.zeros((), dtype=i32, device=dev)
        self._scratch = torch.empty(ops.kv_fork_scratch_size(dec.batch, self.tables.shape[1], dec.n_blocks),
                                    dtype=torch.uint8, device=dev)

    def close(self):
        """Give the decoder its block table back; the pool is not used after it."""
        self.tables.copy_(self._before)

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def fork(self, parents: torch.Tensor | None = None, reserve: torch.Tensor | None = None):
        """Rows become children of `parents` (default: themselves) with room for `reserve` more tokens."""
        d = self.dec
        ops.kv_fork(d.k_arena, d.v_arena, d.cfg.n_layer, self.tables, self.lens, self.pages, self.refs,
                    self.identity if parents is None else parents, reserve=reserve, fill_page=0,
                    status=self._status, scratch=self._scratch)
        self.short = torch.where(self.short == 0, self._status, self.short)

    def compact(self, base: torch.Tensor, path: torch.Tensor, path_lens: torch.Tensor):
        """Keep the accepted branches: base tokens before the draft, path in drafted tokens."""
        d = self.dec
        ops.kv_compact(d.k_arena, d.v_arena, d.cfg.n_layer, self.tables, base, path, path_lens, self.lens)

    def check(self):
        """Raise if a fork so far found too few blocks or bad input (it then changed nothing): what the
        first such fork said."""
        n = int(self.short)
        if n < 0:
            raise ValueError("a fork met a parent, length or block that is out of range")
        if n:
            raise MemoryError(f"the KV arena is {n} blocks short")


class BeamSearcher:
    """Beam search over the captured decode step: the decoder's rows are groups of n_beams beams, and
    every step selects on the device (beam_select) and forks the cache rows after the selected parents
    (kv_fork: shared blocks, one partial block copied per extra child)."""

    def __init__(self, dec: Decoder, n_beams: int, eos: int | None = None):
        if n_beams < 1 or dec.batch % n_beams:
            raise ValueError(f"{dec.batch} decoder rows are not whole groups of {n_beams} beams")
        self.dec, self.n_beams, self.eos = dec, n_beams, eos

    def search(self, prompts, max_new: int):
        """The n_beams best continuations of each prompt, best first: lists of (score, tokens), score the
        sum of the tokens' log-probabilities; a continuation ends at eos (included) or max_new tokens.
        Fewer, if the logits allow fewer."""
        dec, nb = self.dec, self.n_beams
        G, B = len(prompts), dec.batch
        if not 0 < G <= B // nb:
            raise ValueError(f"1 to {B // nb} prompts fit")
        if max_new < 1 or any(not p or len(p) + max_new > dec.max_ctx for p in prompts):
            raise ValueError(f"need non-empty prompts, max_new >= 1 and at most {dec.max_ctx} positions")
        check_tokens(prompts, dec.cfg.vocab)
        with PagePool(dec) as pool:
            return self._search(pool, prompts, max_new)

    def _search(self, pool, prompts, max_new):
        dec, nb = self.dec, self.n_beams
        G, B, dev, i32 = len(prompts), dec.batch, dec.device, torch.int32
        first = torch.arange(G, dtype=i32, device=dev) * nb
        room = torch.zeros(B, dtype=i32, device=dev)
        room[first.long()] = torch.tensor([len(p) for p in prompts], dtype=i32, device=dev)
        pool.fork(reserve=room)
        pool.check()
        _, logits = dec.prefill([g * nb for g in range(G)], prompts)
        pool.lens.copy_(room)
        one = torch.ones(B, dtype=i32, device=dev)
        scores = torch.full((B,), -float("inf"), device=dev)
        parents = torch.full((B,), -1, dtype=i32, device=dev)
        tokens = torch.full((B,), -1, dtype=i32, device=dev)
        s, r, t = ops.beam_select(logits, torch.zeros(G, device=dev), 1, nb)
        scores[:G * nb], tokens[:G * nb] = s.flatten(), t.flatten()
        parents[:G * nb] = torch.where(r >= 0, r * nb, r).flatten()
        finished = torch.zeros(B, dtype=torch.uint8, device=dev)
        eos = -1 if self.eos is None else self.eos
        steps = [(parents.clone(), tokens.clone())]
        out = tuple(torch.empty((B // nb, nb), dtype=d, device=dev) for d in (torch.float32, i32, i32))
        ws = torch.empty(ops.beam_select_scratch_size(B // nb, nb, dec.cfg.vocab, nb), dtype=torch.uint8, device=dev)
        for _ in range(max_new - 1):
            finished.copy_((tokens == eos) & (parents >= 0) if self.eos is not None else finished)
            if bool(((finished != 0) | (parents < 0)).all()):
                break
            pool.fork(parents, reserve=one)
            dec.tokens.copy_(tokens.clamp(min=0))
            dec.ctx_lens.copy_(pool.lens + 1)
            dec.replay()
            pool.lens.add_((parents >= 0).int())
            ops.beam_select(dec.logits, scores, nb, nb, finished=finished, eos=eos, out=out, scratch=ws)
            scores.copy_(out[0].flatten())
            parents.copy_(out[1].flatten())
            tokens.copy_(out[2].flatten())
            steps.append((parents.clone(), tokens.clone()))
        pool.check()
        return beam_paths(scores.tolist(), [(p.tolist(), t.tolist()) for p, t in steps], nb, G, self.eos)


def beam_paths(scores, steps, n_beams: int, groups: int, eos: int | None):
    """(score, tokens) of every live beam, read back through the steps' (parents, tokens)."""
    found = []
    for g in range(groups):
        mine = []
        for row in range(g * n_beams, (g + 1) * n_beams):
            if scores[row] == -float("inf"):
                continue
            out, at = [], row
            for parents, tokens in reversed(steps):
                out.append(tokens[at])
                at = parents[at]
            out.reverse()
            if eos is not None and eos in out:
                out = out[:out.index(eos) + 1]
            mine.append((scores[row], out))
        found.append(mine)
    return found


def ngram_draft(history, n: int = 2, depth: int = 4, width: int = 4):
    """Guess what follows `history` from what followed its last n tokens before: a tree of up to `width`
    different continuations of up to `depth` tokens, latest first.  (tokens, parents), parents as
    Decoder.verify_tree's; -1 = after the last token of the history."""
    tokens, parents, kids = [], [], {}
    key = history[-n:]
    found = 0
    for at in range(len(history) - n - 1, -1, -1):
        if found == width:
            break
        if history[at:at + n] != key:
            continue
        cur, grew = -1, False
        for t in history[at + n:at + n + depth]:
            nxt = kids.get((cur, t))
            if nxt is None:
                nxt = kids[(cur, t)] = len(tokens)
                tokens.append(t)
                parents.append(cur)
                grew = True
            cur = nxt
        found += grew
    return tokens, parents


def accept_path(tokens, parents, greedy):
    """The drafted tokens that greedy decoding would have chosen: token 0 is the last known one, then
    from token to child while a child is what the model says.  Drafted indexes, ascending."""
    path = [0]
    while True:
        nxt = [j for j in range(path[-1] + 1, len(tokens)) if parents[j] == path[-1] and tokens[j] == greedy[path[-1]]]
        if not nxt:
            return path
        path.append(nxt[0])


class TreeSpeculator:
    """Greedy decoding with drafted token trees: `draft(history)` guesses continuations, one pass scores
    the whole tree (Decoder.verify_tree), and the longest branch that greedy decoding would have taken
    is kept (kv_compact).  The tokens are those of greedy decoding."""

    def __init__(self, dec: Decoder, draft=ngram_draft, max_nodes: int = 64):
        if not 1 <= max_nodes <= 1024:
            raise ValueError("max_nodes must be in 1 .. 1024")
        self.dec, self.draft, self.max_nodes = dec, draft, max_nodes
        self.passes = self.accepted = 0

    def generate(self, prompts, max_new: int, eos: int | None = None):
        """The greedy continuation of each prompt (at most max_new tokens, up to eos included)."""
        dec = self.dec
        n, B = len(prompts), dec.batch
        if not 0 < n <= B:
            raise ValueError(f"1 to {B} prompts fit")
        if max_new < 1 or any(not p or len(p) + max_new > dec.max_ctx for p in prompts):
            raise ValueError(f"need non-empty prompts, max_new >= 1 and at most {dec.max_ctx} positions")
        check_tokens(prompts, dec.cfg.vocab)
        with PagePool(dec) as pool:
            return self._generate(pool, prompts, max_new, eos)

    def _generate(self, pool, prompts, max_new, eos):
        dec, n = self.dec, len(prompts)
        B, dev, i32 = dec.batch, dec.device, torch.int32

        def per_row(values, other=0):
            return torch.tensor(list(values) + [other] * (B - n), dtype=i32).to(dev)

        def blocks(tokens):
            return -(-tokens // KV_BLOCK)

        pool.fork(reserve=per_row(len(p) for p in prompts))
        pool.check()
        nxt, _ = dec.prefill(list(range(n)), prompts)
        pool.lens.copy_(per_row(len(p) for p in prompts))
        cached = [len(p) for p in prompts]
        out = [[int(t)] for t in nxt.tolist()]

        def done(i):
            return len(out[i]) >= max_new or (eos is not None and out[i][-1] == eos)

        while True:
            live = [i for i in range(n) if not done(i)]
            if not live:
                return out
            # No row shares blocks, so the host knows how many are free once the finished rows have given theirs
            # back.  Every row's known token comes first (a row without a block for it waits for others to finish),
            # the drafts share what is left.
            free = dec.n_blocks - 1 - sum(blocks(cached[i]) for i in live)
            going = []
            for i in live:
                need = blocks(cached[i] + 1) - blocks(cached[i])
                if need <= free:
                    going.append(i)
                    free -= need
            if not going:
                raise MemoryError(f"no block of the KV arena is free for any of {len(live)} sequences")
            trees = {}
            for i in going:
                t, p = self.draft(list(prompts[i]) + out[i])
                # token 0 is the one just chosen; every drafted token takes a slot of the cache
                least = blocks(cached[i] + 1)
                room = min(self.max_nodes, dec.max_ctx - cached[i], (least + free) * KV_BLOCK - cached[i]) - 1
                trees[i] = ([out[i][-1]] + list(t)[:room], [-1] + [q + 1 for q in list(p)[:room]])
                free -= blocks(cached[i] + len(trees[i][0])) - least
            pool.fork(per_row((i if i in live else -1 for i in range(n)), -1),
                      reserve=per_row(len(trees[i][0]) if i in trees else 0 for i in range(n)))
            pool.check()
            greedy, _ = dec.verify_tree(going, [trees[i] for i in going], [cached[i] for i in going])
            greedy = greedy.tolist()
            paths, at = [[] for _ in range(n)], 0
            base = [cached[i] if i in live else 0 for i in range(n)]
            for i in going:
                t, p = trees[i]
                g = greedy[at:at + len(t)]
                at += len(t)
                path = accept_path(t, p, g)
                new = [t[j] for j in path[1:]] + [g[path[-1]]]
                if eos is not None and eos in new:
                    new = new[:new.index(eos) + 1]
                new = new[:max_new - len(out[i])]
                paths[i] = path
                out[i] += new
                cached[i] += len(path)
                self.accepted += len(new)
            width = max(len(p) for p in paths)
            table = torch.tensor([p + [0] * (width - len(p)) for p in paths] + [[0] * width] * (B - n), dtype=i32).to(dev)
            pool.compact(per_row(base), table, per_row(len(p) for p in paths))
            self.passes += 1
