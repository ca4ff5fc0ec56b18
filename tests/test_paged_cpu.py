"""Refusals of the paged-serving entry points: the C ABI checks its arguments on the host, before any device
work, and the Python calls take CUDA tensors only (no GPU needed here)."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def L():
    from tritiercache_b200.csrc import build
    build.build()
    from tritiercache_b200 import _lib
    return _lib.lib()


A = 0x7000000000  # an address that is never used: each call below is refused, or has nothing to do

TABLES = dict(ctx_lens=A, new_lens=A, tables=A, free_pages=A, free_count=A, free_count_out=A, seq_lens=A, cu_new=A, slots=A,
              positions=A, row_seq=A, row_lens=A, deferred=A, workspace=0, table_stride=8, num_seqs=4, table_width=8,
              free_capacity=64, page_size=16, num_rows=4, position_offset=0)
ROPE = dict(q=A, k=A, v=A, q_out=A, k_dst=A, v_dst=A, q_weight=A, k_weight=A, cos=A, sin=A, positions=A, slots=0,
            q_row_stride=512, q_head_stride=128, k_row_stride=128, k_head_stride=128, v_row_stride=128, v_head_stride=128,
            q_out_row_stride=512, q_out_head_stride=128, k_page_stride=128, k_token_stride=0, k_dst_head_stride=128,
            v_page_stride=128, v_token_stride=0, v_dst_head_stride=128, cos_stride=64, sin_stride=64, table_rows=10, num_pages=0,
            num_rows=3, num_q_heads=4, num_kv_heads=1, head_dim=128, rot_dim=128, page_size=1, dtype=1, q_dtype=1, kv_dtype=1,
            weight_dtype=1, table_dtype=0, positions_i64=0, eps=1e-6, reserved=0)
ATTN = dict(q=A, k=A, v=A, out=A, prefix_table=A, tables=A, row_lens=A, row_seq=0, workspace=A, q_row_stride=512,
            q_head_stride=128, out_row_stride=512, out_head_stride=128, k_page_stride=2048, k_token_stride=128,
            k_head_stride=128, v_page_stride=2048, v_token_stride=128, v_head_stride=128, table_stride=4, num_rows=3,
            num_q_heads=4, num_kv_heads=1, head_dim=128, page_size=16, num_pages=20, prefix_len=40, table_width=4, num_tables=3,
            dtype=1, scale=0.1, reserved=0)


def pack(kind, **kw):
    from tritiercache_b200 import paged
    base, fmt = {"t": (TABLES, paged._TABLES), "r": (ROPE, paged._ROPE), "a": (ATTN, paged._PREFIX)}[kind]
    assert not set(kw) - set(base)
    return fmt.pack(*{**base, **kw}.values())


def status(L, kind, **kw):
    fn = {"t": L.tt_page_tables, "r": L.tt_qk_norm_rope, "a": L.tt_shared_prefix_attention}[kind]
    return fn(pack(kind, **kw), None)


BAD, UNSUPPORTED = 1, 6


@pytest.mark.parametrize("kind,want,kw", [
    ("t", BAD, dict(num_seqs=-1)), ("t", BAD, dict(num_rows=-1)), ("t", BAD, dict(free_capacity=-1)),
    ("t", BAD, dict(page_size=0)), ("t", BAD, dict(table_stride=7)), ("t", BAD, dict(free_count=0)),
    ("t", BAD, dict(ctx_lens=0)), ("t", BAD, dict(tables=0)), ("t", BAD, dict(slots=0)), ("t", BAD, dict(row_lens=0)),
    ("t", BAD, dict(deferred=0)), ("t", UNSUPPORTED, dict(table_width=1 << 20, table_stride=1 << 20, page_size=1 << 11)),
    ("t", BAD, dict(num_rows=100000)),               # needs a workspace
    ("t", BAD, dict(num_seqs=5000, workspace=A + 4)),
    ("r", BAD, dict(num_rows=-1)), ("r", BAD, dict(num_q_heads=0)), ("r", BAD, dict(num_kv_heads=0)),
    ("r", UNSUPPORTED, dict(head_dim=127)), ("r", UNSUPPORTED, dict(head_dim=514)), ("r", BAD, dict(rot_dim=130)),
    ("r", BAD, dict(rot_dim=63)), ("r", BAD, dict(q=0)), ("r", BAD, dict(k_dst=0)), ("r", BAD, dict(cos=0)),
    ("r", BAD, dict(v_dst=0)), ("r", BAD, dict(v=0)), ("r", UNSUPPORTED, dict(dtype=3)), ("r", UNSUPPORTED, dict(q_dtype=2)),
    ("r", UNSUPPORTED, dict(weight_dtype=2)), ("r", UNSUPPORTED, dict(dtype=0)), ("r", BAD, dict(slots=A, page_size=0)),
    ("r", BAD, dict(positions=0, table_rows=2)),
    ("a", BAD, dict(num_rows=-1)), ("a", BAD, dict(num_q_heads=3, num_kv_heads=2)), ("a", UNSUPPORTED, dict(head_dim=96)),
    ("a", UNSUPPORTED, dict(head_dim=256)), ("a", UNSUPPORTED, dict(dtype=0)), ("a", UNSUPPORTED, dict(page_size=8)),
    ("a", UNSUPPORTED, dict(page_size=48)), ("a", BAD, dict(prefix_len=-1)), ("a", BAD, dict(num_tables=2)),
    ("a", BAD, dict(scale=float("nan"))), ("a", BAD, dict(scale=float("inf"))), ("a", UNSUPPORTED, dict(k_token_stride=132)),
    ("a", UNSUPPORTED, dict(v_page_stride=2052)), ("a", UNSUPPORTED, dict(q_head_stride=129)), ("a", UNSUPPORTED, dict(k=A + 8)),
    ("a", UNSUPPORTED, dict(q=A + 2)), ("a", BAD, dict(prefix_table=0)), ("a", BAD, dict(row_lens=0)), ("a", BAD, dict(out=0)),
    ("a", BAD, dict(tables=0)), ("a", UNSUPPORTED, dict(num_rows=1 << 25, row_seq=A)), ("a", UNSUPPORTED, dict(table_width=1 << 28)),
])
def test_bad_arguments_are_refused_on_the_host(L, kind, want, kw):
    assert status(L, kind, **kw) == want, L.tt_last_error()
    assert len(L.tt_last_error()) > 10


def test_null_arguments_and_empty_calls(L):
    for fn in (L.tt_page_tables, L.tt_qk_norm_rope, L.tt_shared_prefix_attention):
        assert fn(None, None) == BAD
    assert status(L, "r", num_rows=0) == 0 and status(L, "a", num_rows=0) == 0
    n = C.c_size_t(7)
    assert L.tt_shared_prefix_attention_workspace(None, C.byref(n)) == BAD
    assert L.tt_shared_prefix_attention_workspace(pack("a", head_dim=32), C.byref(n)) == UNSUPPORTED
    assert L.tt_page_tables_workspace(4, 4) == 0 and L.tt_page_tables_workspace(5000, 4) > 0


def test_python_calls_want_cuda_tensors():
    from tritiercache_b200 import _C
    z = torch.zeros
    i = lambda n: z(n, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="CUDA"):
        _C.page_tables(i(1), i(1), z((1, 4), dtype=torch.int32), i(4), i(1), 16, i(1), i(2), z(1, dtype=torch.int64), i(1), i(1),
                       i(1), i(1))
    with pytest.raises(ValueError, match="CUDA"):
        _C.qk_norm_rope(z(1, 2, 64), z(1, 1, 64), z(1, 1, 64), None, None, z(1, 2, 64), z(1, 1, 64), z(1, 1, 64))
    with pytest.raises(ValueError, match="CUDA"):
        _C.shared_prefix_attention(z(1, 2, 64), z(1, 16, 1, 64), z(1, 16, 1, 64), None, 0, z((1, 1), dtype=torch.int32), i(1),
                                   z(1, 2, 64))
