"""The branching operators together, as the loops use them: tree verification, speculative greedy
decoding and beam search on tiny models."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(layout, batch, max_ctx, seed=11, **kw):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from densecore_b200.decoder import Decoder
    from densecore_b200.ggml_types import Q4_K, Q8_0
    from test_decoder_gpu import tiny
    cfg = tiny(Q8_0) if layout == "q8_0" else tiny(Q4_K, ("attn_v", "ffn_down"))
    return Decoder(cfg, batch=batch, max_ctx=max_ctx, seed=seed, **kw)


@pytest.mark.parametrize("layout", ["q8_0", "q4_k_m"])
def test_verify_tree_equals_each_branch_alone(layout):
    """Every drafted token's logits are those of its own branch ingested as a plain prompt."""
    prompts = [[7, 300, 11, 5, 9, 100, 200, 301, 4, 4, 4, 17, 18], [42, 43]]
    trees = [([1, 2, 3, 2, 9, 8, 7], [-1, 0, 0, 1, 2, 3, 2]), ([5, 6, 7], [-1, 0, 0])]
    a, b = make(layout, 2, 64), make(layout, 1, 64)
    a.prefill([0, 1], prompts)
    nxt, logits = a.verify_tree([0, 1], trees, [len(p) for p in prompts])
    at = 0
    for prompt, (tok, par) in zip(prompts, trees):
        for j in range(len(tok)):
            branch, i = [], j
            while i >= 0:
                branch.append(tok[i])
                i = par[i]
            _, ref = b.prefill([0], [prompt + branch[::-1]])
            x, y = logits[at + j].double().cpu().numpy(), ref[0].double().cpu().numpy()
            assert np.linalg.norm(x - y) / np.linalg.norm(y) < 2e-3     # the bar of prefill against steps
            assert int(nxt[at + j]) == int(logits[at + j].argmax())
        at += len(tok)


def greedy(layout, prompts, max_new, eos=None):
    from densecore_b200.batching import ContinuousBatcher
    b = ContinuousBatcher(make(layout, len(prompts), 96))
    hs = [b.submit(p, max_new, eos) for p in prompts]
    b.run()
    return [h.out for h in hs]


@pytest.mark.parametrize("layout", ["q8_0", "q4_k_m"])
def test_speculator_gives_the_greedy_tokens(layout):
    """Whatever is drafted -- the truth with wrong siblings, nonsense, nothing, n-grams -- the tokens
    are those of greedy decoding, and true drafts take fewer passes."""
    from densecore_b200.batching import TreeSpeculator
    prompts = [[7, 300, 11], [42] * 17, [500, 1, 2, 3, 4, 5, 6]]
    want = greedy(layout, prompts, 20)
    rng = np.random.default_rng(0)

    def truth(history):
        for p, w in zip(prompts, want):
            if history[:len(p)] == p:
                rest = w[len(history) - len(p):][:5]
        tokens, parents, at = [], [], -1
        for t in rest:
            for wrong in rng.integers(0, 400, 2):
                tokens.append(int(wrong))
                parents.append(at)
            tokens.append(t)
            parents.append(at)
            at = len(tokens) - 1
        return tokens, parents

    def nonsense(history):
        n = int(rng.integers(1, 30))
        return [int(x) for x in rng.integers(0, 400, n)], [int(rng.integers(-1, i)) if i else -1 for i in range(n)]

    passes = {}
    for name, draft in (("truth", truth), ("nonsense", nonsense), ("nothing", lambda h: ([], [])), ("ngram", None)):
        dec = make(layout, 4, 96)
        spec = TreeSpeculator(dec, draft, max_nodes=24) if draft else TreeSpeculator(dec)
        assert spec.generate(prompts, 20) == want, name
        passes[name] = spec.passes
    assert passes["truth"] <= 5 and passes["nothing"] == 19


def test_speculator_stops_at_eos_and_frees_blocks():
    from densecore_b200.batching import TreeSpeculator
    prompts = [[7, 300, 11], [500, 1, 2, 3]]
    eos = greedy("q8_0", prompts, 12)[0][4]
    want = greedy("q8_0", prompts, 12, eos)
    assert TreeSpeculator(make("q8_0", 2, 96)).generate(prompts, 12, eos) == want


def branch_score(dec, prompt, tokens):
    """(sum of log-probabilities of `tokens` after prompt, bound of its error) by plain prefills."""
    score = tol = 0.0
    for i, t in enumerate(tokens):
        _, logits = dec.prefill([0], [prompt + tokens[:i]])
        x = logits[0].double()
        score += float(torch.log_softmax(x, -1)[t])
        tol += 2 * 2e-3 * float(x.norm())       # two logits' worth of the bar of prefill against steps
    return score, tol


@pytest.mark.parametrize("layout,nb", [("q8_0", 4), ("q4_k_m", 3), ("q8_0", 1)])
def test_beam_search(layout, nb):
    """Scores are the branches' own log-probabilities; no beam search by plain prefills finds better
    ones; with one beam the tokens are greedy's."""
    from densecore_b200.batching import BeamSearcher
    prompts = [[7, 300, 11, 5, 9, 100, 200, 301, 4, 4, 4, 17, 18, 19], [42]]
    max_new = 5
    got = BeamSearcher(make(layout, 3 * nb, 48), nb).search(prompts, max_new)
    ref = make(layout, 1, 48)
    for prompt, beams in zip(prompts, got):
        assert len(beams) == nb and len({tuple(t) for _, t in beams}) == nb
        assert all(a[0] >= b[0] for a, b in zip(beams, beams[1:]))
        for score, tokens in beams:
            s, tol = branch_score(ref, prompt, tokens)
            assert len(tokens) == max_new and abs(s - score) <= tol
        plain = [(0.0, [])]
        for _ in range(max_new):
            cands = []
            for s, t in plain:
                _, logits = ref.prefill([0], [prompt + t])
                lp = torch.log_softmax(logits[0].double(), -1)
                v, i = lp.topk(nb)
                cands += [(s + float(a), t + [int(b)]) for a, b in zip(v, i)]
            plain = sorted(cands, reverse=True)[:nb]
        assert beams[0][0] >= plain[0][0] - branch_score(ref, prompt, plain[0][1])[1]
    if nb == 1:
        assert [b[0][1] for b in got] == greedy(layout, prompts, max_new)


def test_beam_search_eos_and_short_arena():
    from densecore_b200.batching import BeamSearcher
    prompts = [[7, 300, 11]]
    plain = BeamSearcher(make("q8_0", 4, 64), 4).search(prompts, 8)[0]
    eos = plain[0][1][2]
    got = BeamSearcher(make("q8_0", 4, 64), 4, eos=eos).search(prompts, 8)[0]
    assert any(t[-1] == eos for _, t in got)
    assert all(eos not in t[:-1] and len(t) <= 8 for _, t in got)
    # five blocks: the idle one, the prompt's, and not enough for four diverging beams of 30 tokens
    small = make("q8_0", 4, 64, seq_tokens=[16, 16, 16, 16])
    with pytest.raises(MemoryError):
        BeamSearcher(small, 4).search([[1] * 15], 40)


def test_fork_then_tree_then_compact_on_shared_rows():
    """A beam fork, a tree on each child, compaction: the children's caches are their own -- every
    row's next logits equal those of its whole text from scratch."""
    from densecore_b200.batching import PagePool
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    dec, ref = make("q8_0", 3, 96), make("q8_0", 1, 96)
    text = [int(x) for x in np.random.default_rng(3).integers(0, 400, 37)]
    pool = PagePool(dec)
    pool.fork(reserve=i32([37, 0, 0]))
    dec.prefill([0], [text])
    pool.lens.copy_(i32([37, 0, 0]))
    pool.fork(i32([0, 0, 0]), reserve=i32([6, 6, 6]))
    trees = [([1, 2, 3, 4], [-1, 0, 0, 2]), ([5, 6, 7, 8, 9], [-1, 0, 1, 0, 3]), ([10], [-1])]
    dec.verify_tree([0, 1, 2], trees, [37, 37, 37])
    paths = [[0, 2, 3], [0, 3, 4], [0]]
    pool.compact(i32([37, 37, 37]), i32([[0, 2, 3], [0, 3, 4], [0, 0, 0]]), i32([3, 3, 1]))
    assert pool.lens.tolist() == [40, 40, 38]
    pool.fork(i32([2, 1, 1]), reserve=i32([1, 1, 1]))       # again: row 0 leaves its branch, row 1 gets a twin
    pool.check()
    kept = [[trees[i][0][j] for j in paths[i]] for i in (2, 1, 1)]
    more = [[20], [21], [22]]
    _, logits = dec.verify_tree([0, 1, 2], [(m, [-1]) for m in more], [37 + len(k) for k in kept])
    for i in range(3):
        _, want = ref.prefill([0], [text + kept[i] + more[i]])
        x, y = logits[i].double().cpu().numpy(), want[0].double().cpu().numpy()
        assert np.linalg.norm(x - y) / np.linalg.norm(y) < 2e-3
    pool.fork(i32([-1, -1, -1]))
    assert pool.refs.tolist() == [1] + [0] * (dec.n_blocks - 1)
