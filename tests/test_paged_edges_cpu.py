"""Refusals of the paged operators at the edges of their arguments' ranges (no GPU needed)."""
import pytest

from test_paged_cpu import L, UNSUPPORTED, status  # noqa: F401

TOP = 2 ** 31 - 1


@pytest.mark.parametrize("prefix", [TOP, TOP - 15, TOP - 126])
@pytest.mark.parametrize("rows", [1, 3])
def test_a_prefix_that_does_not_round_up_is_refused(L, prefix, rows):  # noqa: F811
    # 32 bits do not hold its whole tiles of 128 keys
    assert status(L, "a", prefix_len=prefix, page_size=32768, num_rows=rows, workspace=0) == UNSUPPORTED, L.tt_last_error()
    assert b"prefix_len" in L.tt_last_error()


def test_the_longest_prefix_passes_that_check(L):  # noqa: F811
    # refused for its workspace only, after the plan
    assert status(L, "a", prefix_len=TOP - 127, page_size=32768, workspace=0) == 1 and b"workspace" in L.tt_last_error()
