"""Refusals of the paged operators at the edges of their arguments' ranges (no GPU needed)."""
import ctypes as C

import pytest

from test_paged_cpu import L, UNSUPPORTED, pack, status  # noqa: F401

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


@pytest.mark.parametrize("number", [1e39, -1e39, float("nan"), float("inf"), 10 ** 400, -10 ** 400], ids=lambda x: f"{x:.0e}" if isinstance(x, float) else "huge")
def test_numbers_that_no_float_holds_raise_value_errors(monkeypatch, number):
    import torch
    from tritiercache_b200 import _C, paged
    # no tensor here is on a GPU: what is tested is the packing of the numbers, before any call of the library
    monkeypatch.setattr(paged, "_device", lambda t, name: -1)
    monkeypatch.setattr(paged, "_run", lambda *a: pytest.fail("the call went through"))
    z = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError):
        _C.shared_prefix_attention(z(1, 2, 64), z(1, 16, 1, 64), z(1, 16, 1, 64), None, 0, i(1, 1), i(1), z(1, 2, 64), scale=number)
    if isinstance(number, int):
        with pytest.raises(ValueError):
            _C.qk_norm_rope(z(1, 2, 64), z(1, 1, 64), z(1, 1, 64), None, None, z(1, 2, 64), z(1, 1, 64), z(1, 1, 64), eps=number)


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38, -3e38])
def test_a_scale_whose_base_two_form_is_infinite_is_refused(L, scale):  # noqa: F811
    # scores are kept in powers of two: scale * log2(e); infinity times a score of zero would be NaN
    assert status(L, "a", scale=scale) == 1 and b"scale" in L.tt_last_error()
    n = C.c_size_t()
    assert L.tt_shared_prefix_attention_workspace(pack("a", scale=scale / 2), C.byref(n)) == 0


@pytest.mark.parametrize("kw", [dict(dtype="float32"), dict(dtype="float64"), dict(head_dim=96), dict(head_dim=256),
                                dict(page_size=48), dict(page_size=8), dict(page_size=65536), dict(max_pages=1 << 27, page_size=16),
                                dict(num_pages=0), dict(max_rows=0)])
def test_a_batch_that_could_not_attend_is_refused_when_it_is_made(kw):
    import torch
    from tritiercache_b200 import SharedPrefixBatch
    ok = dict(num_pages=8, page_size=16, num_kv_heads=1, head_dim=64, max_requests=2, max_pages=4, max_rows=2, dtype="bfloat16")
    args = {**ok, **kw}
    args["dtype"] = getattr(torch, args["dtype"])
    with pytest.raises(ValueError):
        SharedPrefixBatch(device="cpu", **args)
