"""Shared-prefix attention where the prefix pass's CTAs take spans of several kv heads or row tiles: the queries are
loaded again, the accumulators start anew and V is cleared behind the prefix's end more than once in a CTA's life."""
import ctypes

import numpy as np
import pytest
import torch

from test_gpu_paged import BF, C_, F16, attend, attn_close, make_attn, poison_tail  # noqa: F401

pytestmark = pytest.mark.gpu

CROSSING = [
    # R, nq, nkv, hd, prefix, longest own, page, type, rows a request, layout
    # rows of heads in one tile of 128: even and odd key tiles
    (8, 96, 96, 128, 2000, 30, 16, BF, 1, "nhd"),
    (8, 96, 96, 64, 2049, 30, 32, F16, 1, "kv"),      # a last key tile of one key
    (20, 100, 50, 128, 3841, 9, 16, F16, 2, "hnd"),   # 31 key tiles
    (100, 40, 40, 128, 16385, 40, 64, BF, 1, "nhd"),
    (32, 32, 32, 128, 32769, 20, 128, F16, 1, "nhd"),
    (64, 40, 40, 64, 16700, 33, 16, BF, 1, "hnd"),
    (40, 149, 149, 64, 1281, 9, 16, BF, 1, "nhd"),    # more kv heads than CTAs: spans over whole ones
    (40, 300, 300, 64, 600, 9, 16, F16, 1, "nhd"),    # spans of one key tile among them
    # tiles of 256
    (130, 96, 96, 128, 1999, 20, 16, F16, 1, "nhd"),
    (256, 32, 8, 128, 16400, 30, 32, BF, 1, "nhd"),
    (140, 96, 96, 64, 3001, 20, 16, BF, 1, "kv"),
    # several row tiles of a kv head: side by side, and one after the other
    (300, 48, 48, 128, 1999, 10, 16, BF, 1, "nhd"),
    (600, 16, 2, 128, 9001, 10, 32, F16, 1, "nhd"),   # 19 row tiles
    (600, 16, 2, 64, 9100, 10, 16, BF, 3, "hnd"),
    (5000, 8, 1, 64, 300, 3, 16, BF, 1, "nhd"),       # more row tiles than CTAs
]


@pytest.mark.parametrize("R,nq,nkv,hd,prefix,most,P,dt,chunk,layout", CROSSING)
def test_spans_across_units_match_the_formula(C_, R, nq, nkv, hd, prefix, most, P, dt, chunk, layout):  # noqa: F811
    from tritiercache_b200 import _lib
    r = np.random.default_rng(R + prefix)
    lens = r.integers(0, most + 1, R)
    lens[:3] = most, 0, 1
    s = make_attn(R + hd, R, nq, nkv, hd, prefix, lens, P, dt, chunk, layout)
    poison_tail(s)
    out = attend(C_, s)
    attn_close(out, s, hd ** -0.5)
    for _ in range(5):
        assert torch.equal(attend(C_, s), out)
    err = ctypes.c_int(-1)
    assert _lib.lib().tt_device_error(0, ctypes.byref(err)) == 0 and err.value == 0
