"""The branching operators at the limits of what their description allows: items that begin and end
anywhere in a CTA's range, logits of any size, buffers that calls share, caches that are full."""
import numpy as np
import pytest
import torch

import branch_ref as R
from test_branch_gpu import check_tree, dev, device_error, make_tree, ops, random_seen, run_tree  # noqa: F401

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
