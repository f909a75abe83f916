"""Further refusals and host logic of the branching operators, decided without a GPU."""
import pytest

from densecore_b200 import _lib
from test_branch_cpu import EINVAL, P, compact


# base_lens, path_lens 8 bytes, path and block_tables 32 at P
@pytest.mark.parametrize("kw", [
    dict(base=4 * P, path=4 * P, bt=4 * P, ctx=P), dict(base=4 * P, path=4 * P, bt=4 * P, ctx=P - 4),
    dict(base=4 * P, plens=4 * P, bt=4 * P, ctx=P + 28), dict(base=4 * P, plens=4 * P, path=4 * P, ctx=P + 28)])
def test_compact_refuses_lengths_that_overlap_what_it_reads(kw):
    assert compact(**kw) == EINVAL
    assert b"overlap" in _lib.load().dcg_last_error()
