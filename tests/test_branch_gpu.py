"""Tree attention, page forking, slot compaction and beam selection on the GPU against their plain
definitions (branch_ref.py)."""
import ctypes

import numpy as np
import pytest
import torch

import branch_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from densecore_b200 import ops as _ops
    return _ops


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def device_error(clear=True):
    from densecore_b200 import _lib
    code = ctypes.c_int(-1)
    assert _lib.load().dcg_device_error(ctypes.byref(code), int(clear)) == 0
    return code.value


# ------------------------------------------------------------------------------------------ trees
def random_seen(rng, ns):
    """Rows of a random tree per sequence: (mask words, visible sets); node 0 hangs under the history."""
    rows, seen = [], []
    words = (max(ns) + 63) // 64
    for n in ns:
        mine = []
        for i in range(n):
            mine.append((mine[rng.integers(i)] if i else set()) | {i})
        seen += mine
        rows += [[sum(1 << (t - 64 * w) for t in m if t // 64 == w) for w in range(words)] for m in mine]
    return np.array(rows, dtype=np.uint64).view(np.int64).reshape(-1, words), seen


def make_tree(rng, ns, ctx, hq, hkv, n_layer, extra=3):
    nblk = [(c + 15) // 16 for c in ctx]
    total = sum(nblk) + extra
    perm = rng.permutation(total).astype(np.int32)
    bt = np.zeros((len(ctx), max(max(nblk), 1)), np.int32)
    o = 0
    for s, nb in enumerate(nblk):
        bt[s, :nb] = perm[o:o + nb]
        o += nb
    ka = rng.standard_normal((total * n_layer, 16, hkv, 128)).astype(np.float16)
    va = rng.standard_normal((total * n_layer, 16, hkv, 128)).astype(np.float16)
    starts = np.concatenate([[0], np.cumsum(ns)]).astype(np.int32)
    q = rng.standard_normal((int(starts[-1]), hq, 128)).astype(np.float32)
    return ka, va, bt, starts, q


def run_tree(ops, q, ka, va, n_layer, layer, bt, starts, ctx, mask, hkv, max_tok, max_ctx=None, **kw):
    return ops.paged_attn_tree(dev(q), dev(ka), dev(va), n_layer, layer, dev(bt), dev(starts),
                               dev(np.array(ctx, np.int32)), dev(mask), hkv, max_tok, max_ctx or max(max(ctx), 1), **kw)


def check_tree(ops, ns, ctx, hq, hkv, n_layer=2, layer=1, seed=0, gain=1.0, edit=None, scale=128 ** -0.5):
    rng = np.random.default_rng(seed)
    ka, va, bt, starts, q = make_tree(rng, ns, ctx, hq, hkv, n_layer)
    q *= np.float32(gain)
    mask, seen = random_seen(rng, ns)
    if edit:
        edit(ka, va, bt, starts, mask, seen)
    out = run_tree(ops, q, ka, va, n_layer, layer, bt, starts, ctx, mask, hkv, max(ns), scale=scale).cpu().numpy()
    clean = [np.nan_to_num(a.astype(np.float32), nan=0.0, posinf=0.0, neginf=0.0) for a in (ka, va)]
    ref, tol = R.tree_attention(q, *clean, n_layer, layer, bt, starts, ctx, seen, hkv, scale)
    assert np.isfinite(out).all()
    assert (np.abs(out - ref) <= tol).all(), float((np.abs(out - ref) / (tol + 1e-30)).max())
    assert device_error() == 0
    return out


@pytest.mark.parametrize("hq,hkv", [(8, 8), (16, 8), (32, 8), (64, 8), (6, 2), (7, 1), (20, 4), (48, 3), (3, 3)])
def test_tree_head_layouts(ops, hq, hkv):
    check_tree(ops, [1, 2, 5, 17, 33], [1, 9, 40, 100, 211], hq, hkv)


@pytest.mark.parametrize("hq,hkv,n", [(8, 8, 16), (8, 8, 17), (8, 8, 32), (8, 8, 33), (16, 8, 8), (16, 8, 9), (16, 8, 16),
                                      (32, 8, 4), (32, 8, 5), (32, 8, 8), (64, 8, 2), (64, 8, 3), (64, 8, 4), (64, 8, 5),
                                      (12, 4, 5), (12, 4, 6), (12, 4, 10), (7, 1, 2), (7, 1, 4), (33, 1, 1), (32, 1, 1)])
def test_tree_few_rows(ops, hq, hkv, n):
    """Around 16 and 32 (token, head) rows per kv head, where the kernels change."""
    check_tree(ops, [n, 1, n], [n, 70, 333], hq, hkv, seed=n)


@pytest.mark.parametrize("n", [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 32, 33, 48, 63, 64])
def test_tree_sizes(ops, n):
    check_tree(ops, [n, 1, n], [n, n + 130, 300], 16, 4, seed=n)


@pytest.mark.parametrize("c", [64, 65, 79, 80, 81, 127, 128, 129, 143, 144, 191, 192, 193, 255, 256, 257, 511, 513, 700])
def test_tree_context_edges(ops, c):
    """Contexts that end at and next to the ends of blocks and of the kernels' key tiles."""
    check_tree(ops, [9, 40], [c, c], 8, 2, n_layer=1, layer=0, seed=c)


def test_tree_wide_masks(ops):
    """More than 64 drafted tokens: masks of three words."""
    check_tree(ops, [130, 5, 64], [150, 300, 64], 4, 2)


def test_tree_many_sequences(ops):
    rng = np.random.default_rng(3)
    ns = rng.integers(1, 12, 70).tolist()
    ctx = [n + int(c) for n, c in zip(ns, rng.integers(0, 90, 70))]
    check_tree(ops, ns, ctx, 4, 2, n_layer=1, layer=0)


@pytest.mark.parametrize("most", [12, 20])
def test_tree_many_sequences_of_many_rows(ops, most):
    """More sequences than the planning CTA has threads, some of them empty: up to 48 and 80 rows per kv head."""
    rng = np.random.default_rng(most)
    ns = rng.integers(0, most + 1, 300).tolist()
    ns[0] = ns[299] = most
    ctx = [n + int(c) for n, c in zip(ns, rng.integers(0, 40, 300))]
    check_tree(ops, ns, ctx, 8, 2, n_layer=1, layer=0)


@pytest.mark.parametrize("hq,hkv,most", [(32, 8, 16), (48, 8, 16), (16, 8, 8), (16, 8, 2)])
def test_tree_ragged_batch(ops, hq, hkv, most):
    """Items that begin and end within one CTA's range, several to a range."""
    rng = np.random.default_rng(hq + most)
    ns = rng.integers(1, most + 1, 24).tolist()
    ns[0] = most
    ctx = [n + int(c) for n, c in zip(ns, rng.integers(0, 600, 24))]
    check_tree(ops, ns, ctx, hq, hkv, n_layer=1, layer=0)


def test_tree_few_rows_some_long(ops):
    """Few rows, but contexts too uneven for one CTA per sequence and kv head."""
    rng = np.random.default_rng(11)
    ns = rng.integers(1, 3, 40).tolist()
    ctx = [n + int(c) for n, c in zip(ns, rng.integers(0, 50, 40))]
    ctx[7], ctx[8], ctx[39] = 1700, 900, 1699
    check_tree(ops, ns, ctx, 16, 8, n_layer=1, layer=0)


@pytest.mark.parametrize("ns", [[3], [40]])
def test_tree_long_context(ops, ns):
    check_tree(ops, ns, [5003], 8, 2, n_layer=1, layer=0)


@pytest.mark.parametrize("gain", [1e-6, 1e-3, 8.0, 3e4])
@pytest.mark.parametrize("ns", [[5], [24]])
def test_tree_query_magnitudes(ops, gain, ns):
    """Queries far from 1: nothing over- or underflows on the way to the scores."""
    check_tree(ops, ns, [100], 8, 2, n_layer=1, layer=0, gain=gain, scale=128 ** -0.5 / max(1.0, gain / 8))


@pytest.mark.parametrize("ns", [[4, 4], [33, 40]])
def test_tree_rows_that_see_nothing(ops, ns):
    """No history and a mask without a bit: zeros; with history the history alone."""
    def edit(ka, va, bt, starts, mask, seen):
        for r in (1, int(starts[1]), int(starts[2]) - 1):
            mask[r] = 0
            seen[r] = set()
    out = check_tree(ops, ns, [ns[0], ns[1] + 20], 8, 2, edit=edit)
    assert not out[1].any() and out[ns[0]].any()


def test_tree_mask_without_the_row_itself(ops):
    def edit(ka, va, bt, starts, mask, seen):
        mask[2, 0] = 1
        seen[2] = {0}
    check_tree(ops, [6], [30], 8, 2, edit=edit)


@pytest.mark.parametrize("ns", [[2, 6], [12, 40]])
def test_tree_ignores_what_nobody_sees(ops, ns):
    """NaN and infinities past each context and in the K of a drafted token that no row sees."""
    def edit(ka, va, bt, starts, mask, seen):
        for s, c in enumerate(ctx):
            for p in range(c, bt.shape[1] * 16):
                if p // 16 <= (c - 1) // 16:
                    ka[bt[s, p // 16] * 2 + 1, p % 16] = np.nan
                    va[bt[s, p // 16] * 2 + 1, p % 16] = np.inf if p % 2 else np.nan
        for r in range(len(seen)):     # drafted token 1 of every sequence
            seen[r] = seen[r] - {1}
            mask[r, 0] &= ~np.int64(2)
        for s, c in enumerate(ctx):
            p = c - ns[s] + 1
            ka[bt[s, p // 16] * 2 + 1, p % 16] = np.nan
            va[bt[s, p // 16] * 2 + 1, p % 16] = np.inf
    ctx = [ns[0] + 3, ns[1] + 35]
    check_tree(ops, ns, ctx, 8, 2, edit=edit)


@pytest.mark.parametrize("nodes", [6, 40])
def test_tree_bad_values_stay_with_the_rows_that_see_them(ops, nodes):
    """A NaN in the V of one drafted token: NaN in the rows that see it (in its kv head), the other
    rows as if that token were zero."""
    rng = np.random.default_rng(8)
    ka, va, bt, starts, q = make_tree(rng, [nodes], [90], 8, 2, 1)
    mask, seen = random_seen(rng, [nodes])
    p = 90 - nodes + 2
    clean = va.copy()
    va[bt[0, p // 16], p % 16, 1, 77] = np.nan
    out = run_tree(ops, q, ka, va, 1, 0, bt, starts, [90], mask, 2, nodes).cpu().numpy()
    ref, tol = R.tree_attention(q, ka, clean, 1, 0, bt, starts, [90], seen, 2, 128 ** -0.5)
    for i in range(nodes):
        for h in range(8):
            if 2 in seen[i] and h >= 4:
                assert np.isnan(out[i, h, 77])
            else:
                assert (np.abs(out[i, h] - ref[i, h]) <= tol[i, h]).all()


@pytest.mark.parametrize("nodes", [4, 12, 30])
def test_tree_bad_values_in_many_sequences(ops, nodes):
    """The same in every second sequence of a batch, at places all over the key tiles."""
    rng = np.random.default_rng(nodes)
    ctx = [nodes + int(c) for c in rng.integers(0, 300, 40)]
    ka, va, bt, starts, q = make_tree(rng, [nodes] * 40, ctx, 8, 2, 1)
    mask, seen = random_seen(rng, [nodes] * 40)
    clean, at = va.copy(), rng.integers(0, nodes, 40)
    for s in range(0, 40, 2):
        p = ctx[s] - nodes + at[s]
        va[bt[s, p // 16], p % 16, 1, 77] = np.nan if s % 4 else np.inf
    out = run_tree(ops, q, ka, va, 1, 0, bt, starts, ctx, mask, 2, nodes).cpu().numpy()
    ref, tol = R.tree_attention(q, ka, clean, 1, 0, bt, starts, ctx, seen, 2, 128 ** -0.5)
    for s in range(40):
        for i in range(nodes * s, nodes * (s + 1)):
            bad = s % 2 == 0 and at[s] in seen[i]
            assert np.isnan(out[i, 4:, 77]).all() if bad else np.isfinite(out[i, 4:]).all()
            heads = slice(0, 4 if bad else 8)
            assert (np.abs(out[i, heads] - ref[i, heads]) <= tol[i, heads]).all()


@pytest.mark.parametrize("n", [1, 12, 50])
def test_tree_chain_is_the_causal_prefill(ops, n):
    rng = np.random.default_rng(5)
    ka, va, bt, starts, q = make_tree(rng, [n], [90], 16, 8, 1)
    mask = ops.tree_masks([i - 1 for i in range(n)]).numpy()
    out = run_tree(ops, q, ka, va, 1, 0, bt, starts, [90], mask, 8, n)
    args = (dev(q), dev(ka), dev(va), 1, 0, dev(bt), dev(starts), dev(np.array([90], np.int32)), 8, n, 90)
    pre = ops.paged_attn_prefill(*args)
    _, tol = R.tree_attention(q, ka, va, 1, 0, bt, starts, [90], [set(range(i + 1)) for i in range(n)], 8, 128 ** -0.5)
    assert (np.abs((out - pre).cpu().numpy()) <= 2 * tol).all()


def test_tree_leaves_other_rows(ops):
    """Rows of q before the first, between and behind the sequences are neither read nor written."""
    rng = np.random.default_rng(6)
    ka, va, bt, _, _ = make_tree(rng, [3, 4], [20, 50], 8, 2, 1)
    q = rng.standard_normal((12, 8, 128)).astype(np.float32)
    q[7:] = np.nan
    starts = np.array([0, 3, 7], np.int32)
    mask, seen = random_seen(rng, [3, 4])
    mask = np.concatenate([mask, np.full((5, 1), -1)])
    out = torch.full((12, 8, 128), 7.0, device="cuda")
    run_tree(ops, q, ka, va, 1, 0, bt, starts, [20, 50], mask, 2, 4, out=out)
    assert bool((out[7:] == 7.0).all())
    ref, tol = R.tree_attention(q[:7], ka, va, 1, 0, bt, starts, [20, 50], seen, 2, 128 ** -0.5)
    assert (np.abs(out[:7].cpu().numpy() - ref) <= tol).all()


@pytest.mark.parametrize("n", [3, 30])
def test_tree_empty_sequence(ops, n):
    """A sequence without drafted tokens in the batch (an idle slot)."""
    check_tree(ops, [n, 0, n], [n + 4, 0, 60], 8, 2)


@pytest.mark.parametrize("n", [2, 40])
def test_tree_bad_indexes_are_left_out(ops, n):
    """A block id out of range counts as zeros, an impossible length leaves the sequence's rows alone;
    both are reported, and the other sequences are right."""
    rng = np.random.default_rng(9)
    ka, va, bt, starts, q = make_tree(rng, [n, n, n], [80, 80, 80], 8, 2, 1)
    mask, seen = random_seen(rng, [n, n, n])
    good = bt.copy()
    bt[0, 1], bt[0, 2] = ka.shape[0], -5
    ka2, va2 = np.concatenate([ka, 0 * ka[:1]]), np.concatenate([va, 0 * va[:1]])
    good[0, 1] = good[0, 2] = ka.shape[0]
    assert device_error() == 0
    out = torch.full(q.shape, 7.0, device="cuda")
    run_tree(ops, q, ka, va, 1, 0, bt, starts, [80, n - 1, 80], mask, 2, n, out=out)
    assert device_error() == 2 and device_error() == 0
    ref, tol = R.tree_attention(q, ka2, va2, 1, 0, good, starts, [80, 80, 80], seen, 2, 128 ** -0.5)
    out = out.cpu().numpy()
    ok = np.r_[0:n, 2 * n:3 * n]
    assert (np.abs(out[ok] - ref[ok]) <= tol[ok]).all()
    assert (out[n:2 * n] == 7.0).all()


def test_tree_far_blocks(ops):
    """Blocks behind the 2^31st element of the arena."""
    rng = np.random.default_rng(10)
    n, total = 20, 140000                       # 140000 blocks x 16384 values
    bt = np.array([[139999, 3, 131073, 139000, 70000]], np.int32)
    ka = torch.zeros((total, 16, 8, 128), dtype=torch.float16, device="cuda")
    va = torch.zeros_like(ka)
    small = [rng.standard_normal((5, 16, 8, 128)).astype(np.float16) for _ in range(2)]
    ka[dev(bt[0]).long()], va[dev(bt[0]).long()] = dev(small[0]), dev(small[1])
    q = rng.standard_normal((n, 16, 128)).astype(np.float32)
    starts = np.array([0, n], np.int32)
    mask, seen = random_seen(rng, [n])
    ref, tol = R.tree_attention(q, *small, 1, 0, np.arange(5)[None], starts, [75], seen, 8, 128 ** -0.5)
    for rows in (n, 1):
        st = np.array([0, rows], np.int32)
        ctx = 75 - n + rows
        out = ops.paged_attn_tree(dev(q[:rows]), ka, va, 1, 0, dev(bt), dev(st), dev(np.array([ctx], np.int32)), dev(mask[:rows]), 8, rows, 80)
        assert (np.abs(out.cpu().numpy() - ref[:rows]) <= tol[:rows]).all()
    del ka, va


@pytest.mark.parametrize("n", [3, 40])
def test_tree_captured_streams_and_repeats(ops, n):
    """Captured and replayed with other inputs, on a side stream, twice at once with workspaces of
    their own: bit for bit the eager call."""
    rng = np.random.default_rng(11)
    ka, va, bt, starts, q = make_tree(rng, [n, 2], [700, 33], 16, 4, 1)
    mask, _ = random_seen(rng, [n, 2])
    a = [dev(x) for x in (q, ka, va, bt, starts, np.array([700, 33], np.int32), mask)]

    def call(x, **kw):
        return ops.paged_attn_tree(x, a[1], a[2], 1, 0, a[3], a[4], a[5], a[6], 4, n, 700, **kw)
    eager = call(a[0])
    other = call(a[0].flip(0).contiguous())
    need = max(1, ops.paged_attn_tree_scratch_size(2, 16, 4, n, 700))
    ws = [torch.empty(need, dtype=torch.uint8, device="cuda") for _ in range(2)]
    x, out = a[0].clone(), torch.empty_like(a[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(x, out=out, scratch=ws[0])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, eager)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(x, out=out, scratch=ws[0])
    x.copy_(a[0].flip(0))
    for _ in range(3):
        g.replay()
    assert torch.equal(out, other)
    x.copy_(a[0])
    torch.cuda.synchronize()
    out2 = torch.empty_like(out)
    for _ in range(5):
        with torch.cuda.stream(side):
            call(a[0], out=out2, scratch=ws[1])
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager) and torch.equal(out2, eager)


@pytest.mark.parametrize("n", [9, 12, 16])
def test_tree_rows_between_few_and_many(ops, n):
    """The cases above with 36, 48 and 64 rows per kv head."""
    test_tree_rows_that_see_nothing(ops, [n, n])
    test_tree_ignores_what_nobody_sees(ops, [n, n - 1])
    test_tree_bad_values_stay_with_the_rows_that_see_them(ops, n)
    test_tree_empty_sequence(ops, n)
    test_tree_bad_indexes_are_left_out(ops, n)
    test_tree_captured_streams_and_repeats(ops, n)
    for gain in (1e-6, 8.0, 3e4):
        test_tree_query_magnitudes(ops, gain, [n])


# ------------------------------------------------------------------------------------------- fork
def random_rows(rng, n, mbs, nb, max_len, share=0.5):
    """Rows that share leading blocks, some blocks held from outside, free ones in between."""
    t = [[int(x) for x in rng.integers(0, nb, mbs)] for _ in range(n)]
    order = [int(b) for b in rng.permutation(np.arange(1, nb))]
    refs = [0] * nb
    refs[0] = 1
    lens, held = [], []
    for i in range(n):
        lens.append(int(rng.integers(0, max_len + 1)))
        used = -(-lens[i] // 16)
        held.append(min(mbs, used + int(rng.integers(0, 2))))
        donor = int(rng.integers(0, i)) if i and rng.random() < share else None
        for j in range(held[i]):
            if donor is not None and j < held[donor] // 2:
                t[i][j] = t[donor][j]
            else:
                t[i][j] = order.pop()
            refs[t[i][j]] += 1
    for b in rng.choice(nb, nb // 10, replace=False):      # held by someone else (a prefix cache)
        if b:
            refs[b] += 1
    return t, refs, lens, held


def run_fork(ops, t, refs, lens, held, parents, reserve, fill=0, n_layer=3, hkv=2, seed=0, bad_arena=None):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    g = torch.Generator(device="cuda").manual_seed(seed)
    k = torch.randn((len(refs) * n_layer, 16, hkv, 128), generator=g, device="cuda").half()
    v = torch.randn((len(refs) * n_layer, 16, hkv, 128), generator=g, device="cuda").half()
    k0, v0 = k.clone(), v.clone()
    bt, rf, ln, hd = i32(t), i32(refs), i32(lens), i32(held)
    status = ops.kv_fork(k, v, n_layer, bt, ln, hd, rf, i32(parents), reserve=i32(reserve) if reserve is not None else None, fill_page=fill)
    want = R.fork(t, refs, lens, held, parents, reserve or [0] * len(t), fill)
    got = (bt.tolist(), rf.tolist(), ln.tolist(), hd.tolist())
    for x, y, name in zip(got, want[:4], ("tables", "refs", "lens", "held")):
        assert x == y, name
    assert status.item() == want[5]
    for src, dst, slots in want[4]:
        for a in (k0, v0):
            a.view(len(refs), n_layer, 16, hkv, 128)[dst, :, :slots] = a.view(len(refs), n_layer, 16, hkv, 128)[src, :, :slots].clone()
    assert torch.equal(k, k0) and torch.equal(v, v0)
    return want


@pytest.mark.parametrize("seed", range(12))
def test_fork_random(ops, seed):
    rng = np.random.default_rng(seed)
    n = int(rng.integers(1, 40))
    t, refs, lens, held = random_rows(rng, n, 9, 700, 120)
    parents = [int(x) for x in rng.integers(-1, n, n)]
    reserve = None if seed % 4 == 0 else [int(x) for x in rng.integers(0, 20, n)]
    assert run_fork(ops, t, refs, lens, held, parents, reserve, hkv=1 + seed % 3, seed=seed)[5] == 0


def test_fork_identity_grows_and_frees(ops):
    t = [[5, 6, 7, 8], [1, 2, 3, 0]]
    refs = [1, 1, 1, 1, 0, 1, 1, 1, 1, 0]
    want = run_fork(ops, t, refs, [20, 48], [4, 3], [0, 1], [0, 1])
    assert want[0][0] == [5, 6, 0, 0] and want[0][1] == [1, 2, 3, 4]


def test_fork_one_row_and_dead_rows(ops):
    run_fork(ops, [[1, 2]], [1, 1, 1, 0], [17], [2], [0], [16])
    want = run_fork(ops, [[1, 2], [3, 0]], [1, 1, 1, 1, 0], [17, 3], [2, 1], [-1, -1], [5, 5])
    assert want[1] == [1, 0, 0, 0, 0] and want[3] == [0, 0]
    run_fork(ops, [[1, 2], [3, 0]], [1, 1, 1, 1, 0], [0, 0], [0, 0], [1, 0], [0, 0])


def test_fork_all_children_of_one(ops):
    """31 copies of one partial block; the last child keeps it."""
    t = [[i + 1, 40 + i] for i in range(32)]
    refs = [1] + [1] * 32 + [0] * 7 + [1] * 32 + [0] * 40
    want = run_fork(ops, t, refs, [23] * 32, [2] * 32, [9] * 32, None)
    assert len(want[4]) == 31 and want[0][31][1] == 49


@pytest.mark.parametrize("edit", ["parent", "negative parent", "len", "held", "block", "negative block", "reserve", "wide"])
def test_fork_bad_input_changes_nothing(ops, edit):
    t, refs, lens, held = [[1, 2, 0], [3, 4, 0]], [1, 1, 1, 1, 1, 0, 0, 0], [20, 30], [2, 2]
    parents, reserve = [1, 1], [0, 0]
    if edit == "parent":
        parents = [1, 2]
    elif edit == "negative parent":
        parents = [-2, 1]
    elif edit == "len":
        lens = [20, 33]
    elif edit == "held":
        held = [4, 2]
    elif edit == "block":
        t[0][1] = 8
    elif edit == "negative block":
        t[1][0] = -1
    elif edit == "reserve":
        reserve = [0, -1]
    else:
        reserve = [0, 30]
    assert run_fork(ops, t, refs, lens, held, parents, reserve)[5] == -1


def test_fork_short_of_blocks_changes_nothing(ops):
    t, refs = [[1, 2], [3, 4], [5, 6]], [1, 1, 1, 1, 1, 1, 1, 0]
    assert run_fork(ops, t, refs, [20, 20, 20], [2, 2, 2], [0, 1, 0], [13, 13, 13])[5] == -1    # wider than the table
    # a copy and three reserved blocks; two given back and one free
    assert run_fork(ops, [r + [0] for r in t], refs, [20, 20, 20], [2, 2, 2], [0, 1, 0], [13, 13, 13])[5] == 1
    assert run_fork(ops, t, refs, [20, 20, 20], [2, 2, 2], [0, 1, 0], None)[5] == 0


def test_fork_many_rows_and_a_large_arena(ops):
    rng = np.random.default_rng(5)
    n = 1500
    t, refs, lens, held = random_rows(rng, n, 7, 40000, 90)
    assert run_fork(ops, t, refs, lens, held, [int(x) for x in rng.integers(-1, n, n)], [1] * n, n_layer=1, hkv=1)[5] == 0


@pytest.mark.parametrize("seed", range(4))
def test_fork_wide_tables(ops, seed):
    """Tables of more entries than one CTA counts by itself, with bad input and too few blocks among them."""
    rng = np.random.default_rng(100 + seed)
    n = [30, 300, 1100, 64][seed]
    t, refs, lens, held = random_rows(rng, n, 9, 15000, 130)
    t = [r + [int(x) for x in rng.integers(-5, 20000, 2200 - len(r))] for r in t]
    parents = [int(x) for x in rng.integers(-1, n, n)]
    want = run_fork(ops, t, refs, lens, held, parents, [1] * n, n_layer=1, hkv=1)
    assert want[5] == 0
    if seed < 2:
        assert run_fork(ops, t, refs, lens, held, parents, [1] * (n - 1) + [40000], n_layer=1, hkv=1)[5] == -1
        assert run_fork(ops, t, refs, lens, held, [0] * n, [9000] * n, n_layer=1, hkv=1)[5] > 0


def test_fork_far_blocks_and_capture(ops):
    """Copies between blocks behind the 2^31st element of the arena, from a captured graph."""
    nb = 140000
    k = torch.zeros((nb, 16, 8, 128), dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    k[135000].normal_()
    v[135000].normal_()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    refs = torch.ones(nb, dtype=torch.int32, device="cuda")
    refs[139998] = 0
    bt, ln, hd, par = i32([[135000], [7]]), i32([9, 0]), i32([1, 0]), i32([0, 0])
    ws = torch.empty(ops.kv_fork_scratch_size(2, 1, nb), dtype=torch.uint8, device="cuda")
    st = i32(5)
    start = [x.clone() for x in (bt, ln, hd, refs)]
    ops.kv_fork(k, v, 1, bt, ln, hd, refs, par, status=st, scratch=ws)
    for x, y in zip((bt, ln, hd, refs), start):
        x.copy_(y)
    k[139998].zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.kv_fork(k, v, 1, bt, ln, hd, refs, par, status=st, scratch=ws)
    g.replay()
    assert st.item() == 0 and bt.tolist() == [[139998], [135000]] and ln.tolist() == [9, 9]
    assert torch.equal(k[139998, :9], k[135000, :9]) and torch.equal(v[139998, :9], v[135000, :9])
    assert not k[139998, 9:].any()
    g.replay()      # every row has its block: row 1 becomes a copy of row 0 again
    assert st.item() == 0 and ln.tolist() == [9, 9] and refs[135000].item() + refs[139998].item() == 2
    del k, v


# ---------------------------------------------------------------------------------------- compact
@pytest.mark.parametrize("hkv,n_layer", [(8, 3), (1, 2), (2, 36), (5, 1)])
def test_compact(ops, hkv, n_layer):
    rng = np.random.default_rng(hkv)
    base = [0, 5, 14, 31, 100, 7]
    paths = [[0, 1, 2], [0, 2, 5, 9, 30], [1], [], list(range(1, 40, 2)), [0] + list(range(3, 30))]
    mbs = 10
    perm = rng.permutation(len(base) * mbs).astype(np.int32).reshape(len(base), mbs)
    ka = rng.standard_normal((len(base) * mbs * n_layer, 16, hkv, 128)).astype(np.float16)
    va = rng.standard_normal(ka.shape).astype(np.float16)
    width = max(map(len, paths))
    path = np.full((len(base), width), -9, np.int32)
    for s, p in enumerate(paths):
        path[s, :len(p)] = p
    kd, vd = dev(ka), dev(va)
    ctx = torch.full((len(base),), -1, dtype=torch.int32, device="cuda")
    ops.kv_compact(kd, vd, n_layer, dev(perm), dev(np.array(base, np.int32)), dev(path),
                   dev(np.array([len(p) for p in paths], np.int32)), ctx)
    for a in (ka, va):
        a = a.reshape(len(base) * mbs, n_layer, 16, hkv, 128)
        for s, p in enumerate(paths):
            for j, t in enumerate(p):
                src, dst = base[s] + t, base[s] + j
                a[perm[s, dst // 16], :, dst % 16] = a[perm[s, src // 16], :, src % 16]
    assert np.array_equal(kd.cpu().numpy().view(np.uint16), ka.view(np.uint16))
    assert np.array_equal(vd.cpu().numpy().view(np.uint16), va.view(np.uint16))
    assert ctx.tolist() == [b + len(p) for b, p in zip(base, paths)]
    assert device_error() == 0


@pytest.mark.parametrize("bad", ["order", "repeat", "early", "length", "past the table", "block", "base"])
def test_compact_bad_rows_stay(ops, bad):
    """The bad row is left as it was and reported; its neighbour is moved."""
    path, plen, base = [[0, 2, 5], [0, 2, 5]], [3, 3], [3, 3]
    bt = np.arange(4, dtype=np.int32).reshape(2, 2)
    if bad == "order":
        path[0] = [0, 5, 2]
    elif bad == "repeat":
        path[0] = [0, 2, 2]
    elif bad == "early":
        path[0] = [-1, 2, 5]
    elif bad == "length":
        plen[0] = 4
    elif bad == "past the table":
        path[0] = [0, 2, 29]
    elif bad == "block":
        bt[0, 0] = 4
    else:
        base[0] = -1
    k = torch.randn((4, 16, 2, 128), device="cuda").half()
    v = torch.randn((4, 16, 2, 128), device="cuda").half()
    k0, v0 = k.clone(), v.clone()
    ctx = torch.full((2,), 99, dtype=torch.int32, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    ops.kv_compact(k, v, 1, dev(bt), i32(base), i32(path), i32(plen), ctx)
    assert device_error() == 2
    assert ctx.tolist() == [99, 6]
    for a in (k0, v0):
        a[2, 4:6] = a[2, torch.tensor([5, 8], device="cuda")]
    assert torch.equal(k, k0) and torch.equal(v, v0)


# ------------------------------------------------------------------------------------------- beam
def check_beam(ops, x, scores, n_beams, k, finished=None, eos=-1, view=None):
    xd = dev(x) if view is None else view
    fd = dev(finished) if finished is not None else None
    s, r, t = ops.beam_select(xd, dev(scores), n_beams, k, finished=fd, eos=eos)
    ref = R.beam(x, scores, n_beams, k, finished, eos)
    assert np.array_equal(r.cpu().numpy(), ref[1]) and np.array_equal(t.cpu().numpy(), ref[2])
    got = s.cpu().numpy().astype(np.float64)
    none = np.isneginf(ref[0])
    assert np.array_equal(none, np.isneginf(got))
    # Score: one rounding to fp32, half a step 2^-24, and the error of lse.  A term exp(d), d = x - max,
    # has an argument off by 2^-24 |d log2 e| (product) + 2^-25 |d| (log2 e itself) and a function off by
    # 2^-22: |d| 2^-23 + 2^-22 of itself at most.  Over the terms' own weights |d| averages at most
    # ln(vocab) < 13: 2^-19.3 + 2^-22; the sums of 16 and 32 terms are trees 8 deep: 8 2^-24.  2^-18 holds all.
    assert (np.abs(got - ref[0])[~none] <= 2.0 ** -18 + 2.0 ** -24 * np.abs(ref[0][~none])).all()


@pytest.mark.parametrize("groups,n_beams,vocab,k", [
    (1, 1, 1, 1), (1, 1, 7, 7), (1, 3, 5, 10), (2, 4, 31, 8), (3, 4, 1000, 4), (1, 4, 4095, 8), (2, 5, 4096, 10),
    (2, 5, 4097, 10), (1, 2, 8193, 64), (5, 3, 50001, 6), (1, 16, 20011, 32), (1, 1, 151936, 1), (2, 4, 151936, 8),
    (1, 7, 128256, 33), (40, 2, 12345, 2), (1, 40, 600, 64)])
def test_beam_random(ops, groups, n_beams, vocab, k):
    rng = np.random.default_rng(vocab + k)
    x = (rng.standard_normal((groups * n_beams, vocab)) * 3).astype(np.float32)
    check_beam(ops, x, -rng.random(groups * n_beams).astype(np.float32) * 5, n_beams, k)


@pytest.mark.parametrize("groups,n_beams,vocab,k", [(1, 16, 60007, 32), (2, 40, 30011, 64), (1, 200, 9001, 8)])
@pytest.mark.parametrize("spread", [False, True])
def test_beam_many_lists_of_one_group(ops, groups, n_beams, vocab, k, spread):
    """Few groups of many parts: more candidates than the merge looks at in one go, the best of them in a
    few of the parts or (spread) one in each."""
    rng = np.random.default_rng(vocab + spread)
    x = rng.standard_normal((groups * n_beams, vocab)).astype(np.float32)
    scores = (rng.standard_normal(groups * n_beams) * (0.01 if spread else 3)).astype(np.float32)
    if spread:
        x = np.minimum(x, 3)
        for r in range(len(x)):
            x[r, rng.integers(0, 4096, vocab // 4096) + 4096 * np.arange(vocab // 4096)] = 8 + rng.random(vocab // 4096)
    check_beam(ops, x, scores, n_beams, k)



def test_beam_strided_rows(ops):
    """Rows that are part of wider ones, at every alignment."""
    rng = np.random.default_rng(2)
    wide = (rng.standard_normal((6, 5003)) * 3).astype(np.float32)
    wd = dev(wide)
    for off in range(5):
        for vocab in (4990, 4991, 4992, 4993):
            check_beam(ops, wide[:, off:off + vocab], np.zeros(6, np.float32), 3, 5, view=wd[:, off:off + vocab])


@pytest.mark.parametrize("kind", ["equal", "ascending", "descending", "two values", "zeros of both signs", "one alive", "spikes"])
@pytest.mark.parametrize("k", [1, 4, 33, 64])
def test_beam_ties_and_orders(ops, kind, k):
    """Ties go to the lower token and the lower row, whatever the order the logits come in."""
    vocab = 9001
    i = np.arange(vocab)
    row = {"equal": 0 * i, "ascending": i * 0.001, "descending": -i * 0.001, "two values": i % 2,
           "zeros of both signs": np.where(i % 3, -0.0, 0.0), "one alive": np.where(i == 4321, 1.0, -np.inf),
           "spikes": np.where(i % 1000 == 7, 9.0, -3.0)}[kind].astype(np.float32)
    check_beam(ops, np.stack([row] * 4), np.zeros(4, np.float32), 2, k)


def test_beam_bad_rows_offer_nothing(ops):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((12, 3001)).astype(np.float32)
    x[1, 17] = np.nan
    x[2, 3000] = np.inf
    x[4] = -np.inf
    x[5, ::2] = -np.inf
    scores = np.zeros(12, np.float32)
    scores[6], scores[7], scores[8] = -np.inf, np.nan, np.inf
    x[9:] = np.nan                          # a group without a candidate
    check_beam(ops, x, scores, 3, 6)


def test_beam_far_logits(ops):
    """Logits far from zero and far apart: no overflow of the exponentials."""
    rng = np.random.default_rng(6)
    x = (rng.standard_normal((6, 2000)) * 100).astype(np.float32)
    x[0] += 3e4
    x[1] -= 3e4
    x[2, 5] = 3e38
    x[3] = -3e38
    x[4, 1:] = -3.4028235e38                # masked with the type's lowest value
    check_beam(ops, x, np.zeros(6, np.float32), 2, 8)


def test_beam_sure_beams_and_equal_beams(ops):
    """Beams whose best token takes nearly all (their scores differ by less than fp32 holds next to 1)
    are ordered by what is left, and rows with equal logits tie however the rows are cut."""
    rng = np.random.default_rng(12)
    vocab = 60013
    x = (rng.standard_normal((8, vocab)) * 2).astype(np.float32)
    for r, gap in enumerate((31.0, 33.0, 32.0, 34.5)):
        x[r, 100 * r + 5] = x[r].max() + gap
    x[5:] = x[4]
    check_beam(ops, x, np.zeros(8, np.float32), 4, 9)
    check_beam(ops, np.repeat(x, 12, 0), np.zeros(96, np.float32), 48, 48)


@pytest.mark.parametrize("k", [1, 3, 8])
def test_beam_finished(ops, k):
    rng = np.random.default_rng(7)
    x = (rng.standard_normal((12, 700)) * 3).astype(np.float32)
    scores = -rng.random(12).astype(np.float32) * 4
    finished = np.array([0, 1, 0, 1, 1, 1, 0, 0, 0, 1, 0, 1], np.uint8)
    x[1] = np.nan                           # a finished row's logits are not looked at
    scores[9] = -np.inf
    check_beam(ops, x, scores, 3, k, finished, eos=11)


def test_beam_captured_and_on_a_side_stream(ops):
    rng = np.random.default_rng(9)
    x = [dev((rng.standard_normal((8, 151936)) * 3).astype(np.float32)) for _ in range(2)]
    scores = dev(-rng.random(8).astype(np.float32))
    eager = [ops.beam_select(y, scores, 4, 8) for y in x]
    buf = x[0].clone()
    ws = torch.empty(ops.beam_select_scratch_size(2, 4, 151936, 8), dtype=torch.uint8, device="cuda")
    out = tuple(torch.empty_like(t) for t in eager[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.beam_select(buf, scores, 4, 8, out=out, scratch=ws)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.beam_select(buf, scores, 4, 8, out=out, scratch=ws)
    for i in (1, 0, 1):
        buf.copy_(x[i])
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, eager[i]))


def test_wrappers_refuse(ops):
    h = torch.zeros((4, 16, 2, 128), dtype=torch.float16, device="cuda")
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    m = torch.zeros((1, 1), dtype=torch.int64, device="cuda")
    q = torch.zeros((1, 4, 128), device="cuda")
    for bad in (dict(q=q.half()), dict(bt=i(2, 4)), dict(mask=m.int()), dict(starts=i(1)), dict(q=q.cpu())):
        a = dict(q=q, k=h, v=h, nl=1, layer=0, bt=i(1, 4), starts=i(2), ctx=i(1), mask=m)
        a.update(bad)
        with pytest.raises(ValueError):
            ops.paged_attn_tree(*a.values(), 2, 1, 16)
    with pytest.raises(ValueError):
        ops.kv_fork(h, h, 1, i(1, 4), i(1), i(1), i(5), i(1))            # reference counts of another arena
    with pytest.raises(ValueError):
        ops.kv_fork(h, h, 3, i(1, 4), i(1), i(1), i(4), i(1))            # not whole blocks
    with pytest.raises(ValueError):
        ops.kv_fork(h, h[:, :, :, ::2], 1, i(1, 4), i(1), i(1), i(4), i(1))
    with pytest.raises(ValueError):
        ops.kv_compact(h, h, 1, i(1, 4), i(1), i(1), i(1), i(1))
    with pytest.raises(Exception, match="overlap"):
        n = i(1)
        ops.kv_compact(h, h, 1, i(1, 4), n, i(1, 1), i(1), n)
    x = torch.zeros((4, 10), device="cuda")
    for a in ((x, torch.zeros(3, device="cuda"), 2, 2), (x, torch.zeros(4, device="cuda"), 3, 2),
              (x.t(), torch.zeros(10, device="cuda"), 2, 2), (x.half(), torch.zeros(4, device="cuda"), 2, 2)):
        with pytest.raises(ValueError):
            ops.beam_select(*a)
    with pytest.raises(Exception, match="1 .. 64"):
        ops.beam_select(x, torch.zeros(4, device="cuda"), 2, 65)
