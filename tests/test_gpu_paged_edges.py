"""The paged operators at the edges of their arguments' ranges."""
import numpy as np
import pytest
import torch

from test_gpu_paged import BF, C_, F16, attend, attn_close, attn_ref, make_attn, same, tables_gpu, tables_ref  # noqa: F401

pytestmark = pytest.mark.gpu

TOP = 2 ** 31 - 1


@pytest.mark.parametrize("B", [9, 2500])  # one launch, two launches
@pytest.mark.parametrize("P", [1, 2, 16])
def test_page_tables_lengths_at_the_top_of_their_type(C_, B, P):  # noqa: F811
    """A request that claims up to 2^31 - 1 tokens and brings more is deferred (with pages of one token the sum needs
    more than 31 bits of pages), its neighbours get theirs."""
    W = 3
    ctx, new = np.zeros(B, np.int32), np.ones(B, np.int32)
    ctx[:7] = [TOP, TOP - 1, 1, TOP, TOP, 2, TOP]
    new[:7] = [1, 1, 1, 7, 0, 1, -1]
    tables = np.arange(B * W, dtype=np.int32).reshape(B, W)
    free = np.arange(B * W, 2 * B * W + 20, dtype=np.int32)
    rows = int(np.maximum(new, 0).sum()) + 3
    count = len(free) - 10
    want = tables_ref(ctx, new, tables, free, count, P, rows, 0)
    assert want["deferred"][0] == 3
    same(tables_gpu(C_, ctx, new, tables, free, count, P, rows, 0), want)
    same(tables_gpu(C_, ctx, new, tables, free, count, P, rows, 0, in_place=True), want)


def test_attention_takes_any_stride_of_a_single_row_or_head(C_):  # noqa: F811
    s = make_attn(60, 1, 8, 2, 128, 300, [20], 16, BF)
    want = attend(C_, s)
    attn_close(want, s, 128 ** -0.5)
    one = s["q"].as_strided(s["q"].shape, (1025, 128, 1))
    assert torch.equal(attend(C_, {**s, "q": one}, out=torch.empty_like(s["q"])), want)
    for prefix in (300, 40000):  # read by the rows, and by a pass of its own
        s = make_attn(61, 5, 1, 1, 64, prefix, [20] * 5, 16, BF)
        want = attend(C_, s)
        attn_close(want, s, 64 ** -0.5)
        one = s["q"].as_strided(s["q"].shape, (64, 67, 1))
        assert torch.equal(attend(C_, {**s, "q": one}, out=torch.empty_like(s["q"])), want)


@pytest.mark.parametrize("dt", [BF, F16])
@pytest.mark.parametrize("where", ["prefix", "own"])
@pytest.mark.parametrize("bits", [0, 20, 25.6, 40])
def test_attention_over_many_keys_far_below_the_largest(C_, dt, where, bits):  # noqa: F811
    """One key `bits` powers of two above 2^18 or 2^20 others, all values 1, so the exact output is 1.  A product below
    2^-25 of a tensor core's accumulator may add nothing to it, while its weight counts in the denominator: that is the
    most that may be lost."""
    P, hd = 1024, 64
    nkv, R, n = (160, 2, 2 ** 18) if where == "prefix" else (1, 300, 2 ** 20)
    k = torch.zeros((2, P, nkv, hd), device="cuda", dtype=dt)
    k[0, 0, :, 0] = 1.0  # the first key of page 0; page 1 holds zeros
    v = torch.ones_like(k)
    q = torch.zeros((R, nkv, hd), device="cuda", dtype=dt)
    q[..., 0] = 1.0
    table = torch.ones(n // P, device="cuda", dtype=torch.int32)
    table[0] = 0
    none = torch.zeros((R, 1), device="cuda", dtype=torch.int32)
    lens = torch.zeros(R, device="cuda", dtype=torch.int32)
    out = torch.zeros_like(q)
    scale = max(bits, 2.0 ** -20) * np.log(2.0)
    if where == "prefix":
        C_.shared_prefix_attention(q, k, v, table, n, none, lens, out, scale=scale)
    else:
        C_.shared_prefix_attention(q, k, v, None, 0, table.expand(R, -1), lens + n, out, scale=scale)
    # the last rounding; the weights' (all of one size, a power of two but for bits = 25.6, where they are lost);
    # what is lost; float32 sums of parts of n numbers, each rounded by 2^-24 of the sum so far
    lim = torch.finfo(dt).eps / 2 + (n * 2.0 ** -bits if bits > 25 else 0) + n / 16 * 2.0 ** -24
    assert float((out.double() - 1).abs().max()) <= lim


@pytest.mark.parametrize("dt", [BF, F16])
@pytest.mark.parametrize("R,prefix", [(3, 40), (60, 1500)])  # the rows read the prefix, and a pass of its own
def test_attention_with_scores_of_minus_infinity(C_, dt, R, prefix):  # noqa: F811
    s = make_attn(62, R, 8, 4, 64, prefix, [40] * R, 16, dt)
    s["q"][..., 0] = 1.0
    s["k"][..., 0][s["k"][..., 1] > 0.5] = float("-inf")  # such keys have no weight
    # as attn_close, with the reach of the other keys
    got = attend(C_, s)
    want, mag, _ = attn_ref(s, 64 ** -0.5)
    finite = s["k"].double().where(s["k"] > float("-inf"), 0.0)
    reach = float(s["q"].double().norm(dim=-1).max() * finite.norm(dim=-1).max()) / 8
    u = torch.finfo(dt).eps / 2
    lim = u * want.abs() + mag * (u + 2 * 64 * 2.0 ** -23 * reach + 2.0 ** -20) * 1.01 + (prefix + 40) * 2.0 ** -22 * (dt == F16)
    assert bool(torch.isfinite(want).all()) and bool(((got.double() - want).abs() <= lim).all())
    s["k"][..., 0] = float("-inf")  # nothing left: zeros, as of a row with nothing to attend
    assert bool((attend(C_, s) == 0).all())
