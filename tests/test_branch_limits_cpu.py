"""Further refusals and host logic of the branching operators, decided without a GPU."""
import pytest

from densecore_b200 import _lib
from test_branch_cpu import EINVAL, P, compact, fork


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
