"""The branching operators at the limits of what their description allows: items that begin and end
anywhere in a CTA's range, logits of any size, buffers that calls share, caches that are full."""
import numpy as np
import pytest
import torch

import branch_ref as R
from test_branching_gpu import greedy, make
from test_branch_gpu import check_beam, dev, device_error, make_tree, ops, random_seen, run_tree  # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------ trees
def repeat_tree(ops, rng, ns, ctx, hq, hkv, times=20):
    """Against the definition, and every repeat bit for bit the first call."""
    ka, va, bt, starts, q = make_tree(rng, ns, ctx, hq, hkv, 1)
    mask, seen = random_seen(rng, ns)
    a = [dev(x) for x in (q, ka, va, bt, starts, np.array(ctx, np.int32), mask)]
    ws = torch.empty(max(1, ops.paged_attn_tree_scratch_size(len(ns), hq, hkv, max(ns), max(ctx))), dtype=torch.uint8, device="cuda")
    flush = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")

    def call():
        return ops.paged_attn_tree(a[0], a[1], a[2], 1, 0, *a[3:], hkv, max(ns), max(ctx), scratch=ws)
    first = call()
    ref, tol = R.tree_attention(q, ka, va, 1, 0, bt, starts, ctx, seen, hkv, 128 ** -0.5)
    assert (np.abs(first.cpu().numpy() - ref) <= tol).all()
    for i in range(times):
        if i % 2:
            flush.fill_(i)                  # K, V and Q from memory in one call, from the cache in the next
        assert torch.equal(call(), first)
    assert device_error() == 0


@pytest.mark.parametrize("hq,hkv,most,seqs", [(16, 2, 16, 150), (20, 2, 40, 60), (16, 2, 4, 300)])
def test_tree_items_of_one_tile(ops, hq, hkv, most, seqs):  # noqa: F811
    """Contexts of up to one key tile, so that every item of a range brings a Q of its own: up to 128 rows
    an item, several row tiles, up to 32 rows."""
    rng = np.random.default_rng(most)
    ns = rng.integers(most - most // 3, most + 1, seqs).tolist()
    repeat_tree(ops, rng, ns, [n + int(c) for n, c in zip(ns, rng.integers(0, 128 - most, seqs))], hq, hkv)


@pytest.mark.parametrize("hq,hkv,most", [(16, 2, 16), (12, 2, 20), (16, 2, 8)])
def test_tree_ranges_that_begin_on_an_items_last_tile(ops, hq, hkv, most):  # noqa: F811
    """Two to four key tiles an item and about two items a range: many ranges begin inside an item."""
    rng = np.random.default_rng(most + 1)
    ns = rng.integers(most // 2 + 1, most + 1, 130).tolist()
    repeat_tree(ops, rng, ns, [n + int(c) for n, c in zip(ns, rng.integers(129, 480, 130))], hq, hkv)


@pytest.mark.parametrize("hq,hkv,nodes,seqs,ctx", [(16, 8, 12, 1, 30000), (16, 2, 16, 74, 500), (8, 1, 5, 140, 400)])
def test_tree_first_units_of_a_range(ops, hq, hkv, nodes, seqs, ctx):  # noqa: F811
    """Three to 13 units a range, the first of them from memory: the order of a CTA's first tiles."""
    rng = np.random.default_rng(seqs)
    repeat_tree(ops, rng, [nodes] * seqs, [ctx + int(c) for c in rng.integers(0, 100, seqs)], hq, hkv, times=40)


@pytest.mark.parametrize("hq,hkv,ns,ctx", [(16, 8, [5, 8, 1], [60, 200, 30]), (16, 8, [5, 8], [2000, 700]), (32, 8, [12, 3], [900, 77]),
                                           (32, 4, [40, 9, 40], [300, 64, 1000])])
def test_tree_in_place(ops, hq, hkv, ns, ctx):  # noqa: F811
    """out = q, in every form of the kernel: bit for bit what it is in a buffer of its own."""
    rng = np.random.default_rng(hq + ns[0])
    ka, va, bt, starts, q = make_tree(rng, ns, ctx, hq, hkv, 1)
    mask, _ = random_seen(rng, ns)
    a = [dev(x) for x in (ka, va, bt, starts, np.array(ctx, np.int32), mask)]
    x = dev(q)
    want = ops.paged_attn_tree(x, a[0], a[1], 1, 0, *a[2:], hkv, max(ns), max(ctx))
    for _ in range(5):
        y = x.clone()
        assert ops.paged_attn_tree(y, a[0], a[1], 1, 0, *a[2:], hkv, max(ns), max(ctx), out=y) is y
        assert torch.equal(y, want)


def test_tree_refuses_another_head_layout(ops):  # noqa: F811
    """kv heads or a head size that the arenas do not have, although the sizes divide."""
    h = torch.zeros((4, 16, 8, 128), dtype=torch.float16, device="cuda")
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    m = torch.zeros((1, 1), dtype=torch.int64, device="cuda")
    q = torch.zeros((1, 8, 128), device="cuda")

    def call(k, v, hkv, q=q):
        return ops.paged_attn_tree(q, k, v, 1, 0, i(1, 4), i(2), i(1), m, hkv, 1, 16)
    for k, v, hkv in ((h, h, 4), (h, h, 1), (h.view(8, 16, 4, 128), h, 4), (h, h.view(2, 16, 16, 128), 8), (h.view(4, 16, 16, 64), h, 8)):
        with pytest.raises(ValueError, match="kv heads"):
            call(k, v, hkv)
    call(h, h, 8)
    call(h.flatten(), h.view(64, 8, 128), 8)     # another form of the same layout


@pytest.mark.parametrize("hq,hkv,nodes", [(8, 2, 3), (8, 2, 7), (8, 2, 12), (16, 2, 12), (32, 2, 30)])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_tree_infinities_stay_with_the_rows_that_see_them(ops, hq, hkv, nodes, bad):  # noqa: F811
    """Infinities in K and V of the history reach the rows of their kv head and sequence, one in a drafted K the
    rows that see it; all others are right, in every form of the kernel."""
    rng = np.random.default_rng(nodes)
    ns, ctx = [nodes] * 4, [nodes + 300, nodes + 40, nodes + 140, nodes + 260]
    ka, va, bt, starts, q = make_tree(rng, ns, ctx, hq, hkv, 1)
    mask, seen = random_seen(rng, ns)
    k0, v0 = ka.copy(), va.copy()
    ka[bt[0, 3], 5, 1, 17] = bad                 # history of sequence 0, kv head 1
    va[bt[2, 0], 2, 0, 99] = bad                 # history of sequence 2, kv head 0
    p = ctx[3] - nodes + 1                       # drafted token 1 of sequence 3, kv head 0
    ka[bt[3, p // 16], p % 16, 0, 3] = bad
    out = run_tree(ops, q, ka, va, 1, 0, bt, starts, ctx, mask, hkv, nodes).cpu().numpy()
    ref, tol = R.tree_attention(q, k0, v0, 1, 0, bt, starts, ctx, seen, hkv, 128 ** -0.5)
    half, checked = hq // 2, 0
    for i in range(len(q)):
        s = i // nodes
        heads = slice(0, half) if s == 0 else slice(half, hq) if s == 2 or (s == 3 and 1 in seen[i]) else slice(0, hq)
        assert (np.abs(out[i, heads] - ref[i, heads]) <= tol[i, heads]).all()
        checked += s == 3 and heads == slice(0, hq)
    assert checked and device_error() == 0


# ------------------------------------------------------------------------------------------- beam
# The bound of check_beam (2^-19.3 + 2^-22 + 8 2^-24 = 2.3 10^-6 of 2^-18 = 3.8 10^-6) holds at any offset M.  Up to
# |M| = 2^24 the one factor more, 2^-l with |l| <= 1, is off by 2^-22, and l adds 2^-24 to the arguments' rounding: 0.3 10^-6.
# From 2^24 on logits that differ do so by 1 at least, x - max is exact and the sums are those of the first case; from
# 2^28 on (steps of 32) only equal logits count, whose sum is exact, and 64-bit lse and score are rounded by 2^-25 |M| 2^-28
# at most on each side: 10^-6 at 2^33, beyond which log(vocab) itself is lost on both sides alike.
@pytest.mark.parametrize("big", [2.0 ** 23, 16777214.0, 2.0 ** 24, 1e9, 5e9, 6e9, 1e10, 1e12, 1e20, 1e30, 9.9e37, 1.1e38, 3e38])
@pytest.mark.parametrize("k", [4, 40])
def test_beam_masked_and_offset_logits(ops, big, k):  # noqa: F811
    """Logits masked with a large finite number (all but a few, whole tiles, the padding of a vocabulary),
    and rows that lie around it."""
    rng = np.random.default_rng(int(np.log2(big)))
    x = (rng.standard_normal((8, 20011)) * 3).astype(np.float32)
    x[0, rng.permutation(20011)[5:]] = -big
    x[1, -267:] = -big
    x[2, 4096:8192] = -big
    x[3, 511:] = -big
    x[4] += np.float32(big)
    x[5] -= np.float32(big)
    x[6, 1:] = -big
    x[7] = np.float32(big) * (1 + rng.integers(0, 3, 20011).astype(np.float32) / 64) * (1 if big < 3e38 else 0.9)
    scores = -rng.random(8).astype(np.float32) * 4
    check_beam(ops, x, scores, 4, k)
    check_beam(ops, x, scores, 1, k)
    check_beam(ops, x, scores, 8, k)


@pytest.mark.parametrize("big", [1e10, 1e20, 3.4028235e38])
def test_beam_padded_vocabulary(ops, big):  # noqa: F811
    rng = np.random.default_rng(13)
    x = (rng.standard_normal((8, 151936)) * 3).astype(np.float32)
    x[:, -267:] = -big
    check_beam(ops, x, -rng.random(8).astype(np.float32) * 4, 4, 8)


def test_beam_scores_in_place(ops):  # noqa: F811
    """out_scores may be scores itself when there are as many results as beams."""
    rng = np.random.default_rng(14)
    x = dev((rng.standard_normal((40, 9001)) * 3).astype(np.float32))
    scores = dev(-rng.random(40).astype(np.float32) * 4)
    want = ops.beam_select(x, scores, 4, 4)
    out = (scores, torch.empty_like(want[1]), torch.empty_like(want[2]))
    ops.beam_select(x, scores, 4, 4, out=out)
    assert torch.equal(scores.view(10, 4), want[0]) and torch.equal(out[1], want[1]) and torch.equal(out[2], want[2])


# ---------------------------------------------------------------------------------- the decode loops
@pytest.mark.parametrize("loop", ["speculator", "beams"])
def test_loops_give_the_decoder_back(loop):
    """A decoder that a loop has used serves direct calls as one that it has not."""
    from densecore_b200.batching import BeamSearcher, TreeSpeculator
    used, fresh = make("q8_0", 4, 96), make("q8_0", 4, 96)
    prompts = [[7, 300, 11] * 6, [42] * 5]
    if loop == "speculator":
        TreeSpeculator(used).generate(prompts, 20)
    else:
        BeamSearcher(used, 2).search(prompts, 20)
    assert torch.equal(used.block_tables, fresh.block_tables)
    texts = [[int(t) for t in np.random.default_rng(i).integers(0, 400, 20 + i)] for i in range(4)]
    for d in (used, fresh):
        nxt, d.seen = d.prefill(range(4), texts)
        d.tokens.copy_(nxt)
        d.ctx_lens.copy_(torch.tensor([len(t) + 1 for t in texts], dtype=torch.int32))
        d.replay()
    assert torch.equal(used.seen, fresh.seen) and torch.equal(used.logits, fresh.logits)


def test_full_caches():
    """Requests that fill the decoder's cache to its last slot, in every loop that hands out blocks."""
    from densecore_b200.batching import BeamSearcher, ContinuousBatcher, TreeSpeculator
    prompts = [[7, 300, 11, 5] * 10, [42, 43] * 20]
    want = greedy("q8_0", prompts, 24)
    assert TreeSpeculator(make("q8_0", 2, 64)).generate(prompts, 24) == want
    b = ContinuousBatcher(make("q8_0", 2, 64))
    hs = [b.submit(p, 24) for p in prompts]
    b.run(200)
    assert [h.out for h in hs] == want and len(b.alloc.free) == b.alloc.n_blocks - 1
    assert [x[0][1] for x in BeamSearcher(make("q8_0", 2, 64), 1).search(prompts, 24)] == want
    # four beams that have nothing but their first token in common
    beams = BeamSearcher(make("q8_0", 4, 48), 4).search([[300]], 47)[0]
    assert len(beams) == 4 and len({tuple(t) for _, t in beams}) == 4 and all(len(t) == 47 for _, t in beams)


def test_decoder_tables_and_history_with_the_idle_block():
    """The idle block lies behind the sequences' own: no table row starts with it, and the random history of
    the others is the one that a seed gives an arena of their size."""
    dec = make("q8_0", 2, 40, seq_tokens=[40, 17])
    assert dec.n_blocks == 3 + 2 + 1 and dec.k_arena.shape[0] == dec.n_blocks * dec.cfg.n_layer
    held = dec.block_tables.cpu()
    assert sorted(held[0].tolist() + held[1, :2].tolist()) == list(range(5))
    dec.fill_kv_random(3)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    for arena in (dec.k_arena, dec.v_arena):
        own = arena[:5 * dec.cfg.n_layer]
        assert torch.equal(own, torch.empty_like(own).normal_(0.0, 1.0, generator=g)) and not arena[5 * dec.cfg.n_layer:].any()


def test_speculator_in_a_tight_arena():
    """An arena that holds the finished texts is enough, whatever is drafted."""
    from densecore_b200.batching import TreeSpeculator
    rng = np.random.default_rng(0)

    def wild(history):
        return [int(x) for x in rng.integers(0, 400, 40)], [int(rng.integers(-1, i)) if i else -1 for i in range(40)]
    prompts = [[7, 300, 11] * 5, [42] * 17, [500, 1, 2]]
    dec = make("q8_0", 3, 96, seq_tokens=[len(p) + 29 for p in prompts])
    spec = TreeSpeculator(dec, wild)
    assert spec.generate(prompts, 30) == greedy("q8_0", prompts, 30)
    assert device_error() == 0


def test_verify_tree_on_two_shards(monkeypatch):
    """The tensor-parallel pass: two shards of a model on this GPU, a thread each, with sums and gathers that
    the host makes (no kernel waits for another), against the whole model."""
    import threading

    import torch.distributed as dist
    from densecore_b200 import _lib
    from densecore_b200.decoder import Decoder
    from test_tp_gpu import _config
    cfg, batch, _, max_ctx = _config("tiny")
    whole = Decoder(cfg, batch=batch, max_ctx=max_ctx, seed=7)
    shards = [Decoder(cfg, batch=batch, max_ctx=max_ctx, seed=7, tp_rank=r, tp_size=2) for r in range(2)]
    meet, given, me = threading.Barrier(2, timeout=60), [None, None], threading.local()

    def exchange(x):
        given[me.rank] = x.clone()
        meet.wait()
        both = [t.clone() for t in given]
        meet.wait()
        return both
    monkeypatch.setattr(dist, "all_reduce", lambda y, group=None: y.copy_(sum(exchange(y))))
    monkeypatch.setattr(dist, "all_gather_into_tensor", lambda out, x, group=None: out.copy_(torch.stack(exchange(x))))
    prompts = [[7, 300, 11, 5, 9, 100, 200, 301, 4, 4, 4, 17, 18], [42, 43]]
    trees = [([1, 2, 3, 2, 9, 8, 7], [-1, 0, 0, 1, 2, 3, 2]), ([5, 6, 7], [-1, 0, 0])]

    def run(dec):
        dec.prefill([0, 1], prompts)
        return dec.verify_tree([0, 1], trees, [len(p) for p in prompts])
    got = [None, None]

    def work(r):
        me.rank = r
        try:
            got[r] = run(shards[r])
        except BaseException as e:   # noqa: BLE001 -- told below; the other thread's barrier runs out
            meet.abort()
            got[r] = e
    prev = _lib.load().dcg_set_programmatic_launch(1)
    threads = [threading.Thread(target=work, args=(r,)) for r in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    _lib.load().dcg_set_programmatic_launch(prev)        # the threads' own saving of it may have crossed
    for g in got:
        if isinstance(g, BaseException):
            raise g
    _, want = run(whole)
    for nxt, logits in got:
        assert torch.equal(logits, got[0][1]) and torch.equal(nxt, logits.argmax(-1))
        x, y = logits.double(), want.double()
        assert bool(((x - y).norm(dim=-1) / y.norm(dim=-1) < 2e-3).all())      # the bar of shards against the whole
