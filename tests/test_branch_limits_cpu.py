"""Further refusals and host logic of the branching operators, decided without a GPU."""
import pytest

from densecore_b200 import _lib
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
