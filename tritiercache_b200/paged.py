"""Paged serving of a batch of requests on a shared prompt (tt_page_tables,
tt_qk_norm_rope, tt_shared_prefix_attention in include/tritier_b200.h).

No reference counterpart: the reference serves one sequence per engine.  The
calls take CUDA tensors in place, run on the current torch stream of the
tensors' device, do not wait for the GPU and may be captured into CUDA graphs.
Bad arguments raise ValueError before any device work.  Lengths, slots,
positions and page numbers live on the device and are not read back; what an
impossible one does is said at each call.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from typing import Optional

import torch

from ._lib import check, lib

_DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_I32, _I64 = torch.int32, torch.int64

# the argument structs of the C ABI, packed with native alignment
_TABLES = struct.Struct("@14Pq6i")
_ROPE = struct.Struct("@12P18q12ifi")
_PREFIX = struct.Struct("@9P11q10ifi")


def _device(t, name: str):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path).")
    return t.device


def _gaps(t) -> bool:
    """Whether neighbours along the last dimension do not lie side by side."""
    return t.shape[-1] > 1 and t.stride(-1) != 1 and t.numel() > 0


def _vec(t, name: str, dev, dtype, n: Optional[int] = None):
    """Address of a contiguous 1-D tensor of `dtype` with n elements (None: any)."""
    if not isinstance(t, torch.Tensor) or t.device != dev:
        raise ValueError(f"{name} must be a tensor on {dev}.")
    if t.dtype != dtype or t.dim() != 1 or (n is not None and t.shape[0] != n) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous {dtype} of shape [{'n' if n is None else n}], got {t.dtype} "
                         f"{tuple(t.shape)}.")
    return t.data_ptr()


def _run(fn, packed: bytes, dev, what: str) -> None:
    if torch.cuda.current_device() == dev.index:
        st = fn(packed, torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(dev):
            st = fn(packed, torch.cuda.current_stream().cuda_stream)
    if st:
        check(st, what)


def page_tables(ctx_lens, new_lens, tables, free_pages, free_count, page_size, seq_lens, cu_new, slots, positions,
                row_seq, row_lens, deferred, free_count_out=None, position_offset=0) -> None:
    """Gives a step's new tokens their pages, slots and positions.

    Request b holds ``ctx_lens[b]`` tokens in the pages of its row of
    ``tables`` [requests, width] and brings ``new_lens[b]`` (0: rests, -1: has
    ended, its pages go back on the stack).  Pages are popped from
    ``free_pages[:free_count]`` in request order; a request that does not fit
    (stack, table width, row buffers) is deferred and its rows are padding.
    Writes tables and free_pages in place, ``free_count_out`` (default:
    free_count itself), ``seq_lens`` [requests] (may be ctx_lens), ``cu_new``
    [requests + 1], per row ``slots`` int64, ``positions`` (ctx + i +
    position_offset), ``row_seq``, ``row_lens`` (-1, 0, -1, 0 for padding), and
    ``deferred`` [1], the number of deferred requests.  All int32 but slots.
    """
    dev = _device(tables, "tables")
    if tables.dtype != _I32 or tables.dim() != 2 or _gaps(tables):
        raise ValueError("tables must be int32 [requests, width] with contiguous rows.")
    B, W = tables.shape
    n = slots.shape[0] if isinstance(slots, torch.Tensor) and slots.dim() == 1 else None
    ps = [_vec(ctx_lens, "ctx_lens", dev, _I32, B), _vec(new_lens, "new_lens", dev, _I32, B), tables.data_ptr(),
          _vec(free_pages, "free_pages", dev, _I32), _vec(free_count, "free_count", dev, _I32, 1),
          _vec(free_count if free_count_out is None else free_count_out, "free_count_out", dev, _I32, 1),
          _vec(seq_lens, "seq_lens", dev, _I32, B), _vec(cu_new, "cu_new", dev, _I32, B + 1),
          _vec(slots, "slots", dev, _I64), _vec(positions, "positions", dev, _I32, n),
          _vec(row_seq, "row_seq", dev, _I32, n), _vec(row_lens, "row_lens", dev, _I32, n),
          _vec(deferred, "deferred", dev, _I32, 1)]
    L = lib()
    size = L.tt_page_tables_workspace(B, n)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    _run(L.tt_page_tables, _TABLES.pack(*ps, 0 if ws is None else ws.data_ptr(), tables.stride(0) if B > 1 else max(W, 1), B, W,
                                        free_pages.shape[0], int(page_size), n, int(position_offset)), dev, "page_tables")


def _heads(t, name: str, dev, dtype, rows, heads, hd):
    if not isinstance(t, torch.Tensor) or t.device != dev:
        raise ValueError(f"{name} must be a tensor on {dev}.")
    if t.dtype != dtype or t.shape != (rows, heads, hd) or _gaps(t):
        raise ValueError(f"{name} must be {dtype} {(rows, heads, hd)} with contiguous channels, got {t.dtype} "
                         f"{tuple(t.shape)}, strides {tuple(t.stride())}.")
    return t.data_ptr()


def _apart(t, name: str) -> None:
    """An output whose dimensions overlap (an expanded one) would be written by several threads."""
    for n, st in zip(t.shape, t.stride()):
        if n > 1 and st == 0:
            raise ValueError(f"{name} is an output and must not be an expanded tensor.")


def _pool(t, name: str, dev, dtype, heads, hd):
    if not isinstance(t, torch.Tensor) or t.device != dev:
        raise ValueError(f"{name} must be a tensor on {dev}.")
    if t.dtype != dtype or t.dim() != 4 or t.shape[2] != heads or t.shape[3] != hd or _gaps(t):
        raise ValueError(f"{name} must be {dtype} [pages, page_size, {heads}, {hd}] with contiguous channels, got {t.dtype} "
                         f"{tuple(t.shape)}, strides {tuple(t.stride())}.")
    return t.data_ptr()


def qk_norm_rope(q, k, v, cos, sin, q_out, k_dst, v_dst, q_weight=None, k_weight=None, eps=1e-6, positions=None,
                 slots=None) -> None:
    """RMS norm of every query and key head (where its weight is given),
    rotate-half rotation by position, and the placing of q, k and v, in one pass.

    ``q`` [rows, q_heads, head_dim], ``k``, ``v`` [rows, kv_heads, head_dim], any
    row and head strides (parts of a fused projection).  ``cos``/``sin``
    [table rows, rot_dim / 2], row ``positions[i]`` (int32 or int64; None: i)
    belongs to row i; channels from rot_dim on are not rotated; None: no
    rotation.  ``q_out`` [rows, q_heads, head_dim]; ``k_dst``/``v_dst`` are dense
    [rows, kv_heads, head_dim], or with ``slots`` (int64, distinct) pools
    [pages, page_size, kv_heads, head_dim].  Outputs have the inputs' type or
    float32; weights and tables likewise.  ``v`` and ``v_dst`` may be None.
    Rows with a slot outside the pool (-1: padding) are left as they are in
    every output; a position outside the tables makes the rotated channels NaN.
    q_out may be q itself, dense k_dst and v_dst k and v.
    """
    dev = _device(q, "q")
    dt = q.dtype
    if dt not in _DT or q.dim() != 3:
        raise ValueError("q must be float32, bfloat16 or float16 [rows, heads, head_dim].")
    R, nq, hd = q.shape
    if not isinstance(k, torch.Tensor) or k.dim() != 3:
        raise ValueError("k must be a tensor [rows, kv_heads, head_dim].")
    nkv = k.shape[1]
    for t, name in ((q_out, "q_out"), (k_dst, "k_dst")):
        if not isinstance(t, torch.Tensor) or t.dtype not in (dt, torch.float32):
            raise ValueError(f"{name} must be a tensor of {dt} or float32.")
        _apart(t, name)
    if (v is None) != (v_dst is None):
        raise ValueError("v and v_dst come together.")
    if v_dst is not None:
        if not isinstance(v_dst, torch.Tensor):
            raise ValueError("v_dst must be a tensor.")
        _apart(v_dst, "v_dst")
    kt = k_dst.dtype
    pq, pk, po = _heads(q, "q", dev, dt, R, nq, hd), _heads(k, "k", dev, dt, R, nkv, hd), _heads(q_out, "q_out", dev, q_out.dtype, R, nq, hd)
    pv = 0 if v is None else _heads(v, "v", dev, dt, R, nkv, hd)
    if slots is None:
        pkd = _heads(k_dst, "k_dst", dev, kt, R, nkv, hd)
        pvd = 0 if v is None else _heads(v_dst, "v_dst", dev, kt, R, nkv, hd)
        psl, pages, psize = 0, R, 1
        kst = (k_dst.stride(0), 0, k_dst.stride(1))
        vst = (0, 0, 0) if v is None else (v_dst.stride(0), 0, v_dst.stride(1))
    else:
        pkd = _pool(k_dst, "k_dst", dev, kt, nkv, hd)
        pvd = 0
        if v is not None:
            pvd = _pool(v_dst, "v_dst", dev, kt, nkv, hd)
            if v_dst.shape != k_dst.shape:
                raise ValueError("k_dst and v_dst must have the same shape.")
        psl, pages, psize = _vec(slots, "slots", dev, _I64, R), k_dst.shape[0], k_dst.shape[1]
        kst = k_dst.stride()[:3]
        vst = (0, 0, 0) if v is None else v_dst.stride()[:3]
    wt = tt = dt
    pw = [0, 0]
    for i, (w, name) in enumerate(((q_weight, "q_weight"), (k_weight, "k_weight"))):
        if w is not None:
            if not isinstance(w, torch.Tensor) or w.dtype not in (dt, torch.float32):
                raise ValueError(f"{name} must be a tensor of {dt} or float32.")
            wt = w.dtype
            pw[i] = _vec(w, name, dev, wt, hd)
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError("q_weight and k_weight must have the same type.")
    pc = psn = cst = sst = trows = rot = 0
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together.")
    if cos is not None:
        if not isinstance(cos, torch.Tensor) or cos.dim() != 2 or cos.dtype not in (dt, torch.float32):
            raise ValueError(f"cos must be {dt} or float32 [table rows, rot_dim / 2].")
        tt, trows, rot = cos.dtype, cos.shape[0], 2 * cos.shape[1]
        for t, name in ((cos, "cos"), (sin, "sin")):
            if not isinstance(t, torch.Tensor) or t.device != dev or t.dtype != tt or t.shape != cos.shape or \
                    _gaps(t):
                raise ValueError(f"{name} must be {tt} {tuple(cos.shape)} on {dev} with contiguous rows.")
        pc, psn, cst, sst = cos.data_ptr(), sin.data_ptr(), cos.stride(0), sin.stride(0)
        if rot == 0:
            pc = psn = 0
    ppos, p64 = 0, 0
    if positions is not None:
        p64 = 1 if isinstance(positions, torch.Tensor) and positions.dtype == _I64 else 0
        ppos = _vec(positions, "positions", dev, _I64 if p64 else _I32, R)
    if R == 0:
        return
    packed = _ROPE.pack(pq, pk, pv, po, pkd, pvd, pw[0], pw[1], pc, psn, ppos, psl, q.stride(0), q.stride(1), k.stride(0),
                        k.stride(1), v.stride(0) if pv else 0, v.stride(1) if pv else 0, q_out.stride(0), q_out.stride(1),
                        *kst, *vst, cst, sst, trows, pages, R, nq, nkv, hd, rot, psize, _DT[dt], _DT[q_out.dtype], _DT[kt],
                        _DT[wt], _DT[tt], p64, float(eps), 0)
    _run(lib().tt_qk_norm_rope, packed, dev, "qk_norm_rope")


def shared_prefix_attention(q, k_pages, v_pages, prefix_table, prefix_len, tables, row_lens, out, row_seq=None,
                            scale=None) -> None:
    """Decode attention of a batch over a prefix that all rows share, read once
    for all of them, and over each row's own pages.

    ``q``, ``out`` [rows, q_heads, head_dim]; ``k_pages``/``v_pages`` [pages,
    page_size, kv_heads, head_dim] (any strides that keep channels contiguous and
    16-byte steps; bfloat16 or float16 throughout).  Row r attends tokens
    [0, prefix_len) of the pages in ``prefix_table`` and tokens [0, row_lens[r])
    of the pages in row ``row_seq[r]`` (None: r) of ``tables``.  ``scale``
    defaults to head_dim ** -0.5.  Rows with row_seq < 0 are padding and stay as
    they were; a row with nothing to attend gives zeros; a page outside the pool
    or a length beyond the table gives NaN.  out may be q itself.
    """
    dev = _device(q, "q")
    dt = q.dtype
    if dt not in (torch.bfloat16, torch.float16) or q.dim() != 3:
        raise ValueError("q must be bfloat16 or float16 [rows, heads, head_dim].")
    R, nq, hd = q.shape
    if not isinstance(k_pages, torch.Tensor) or k_pages.dim() != 4:
        raise ValueError("k_pages must be a tensor [pages, page_size, kv_heads, head_dim].")
    nkv = k_pages.shape[2]
    pq, po = _heads(q, "q", dev, dt, R, nq, hd), _heads(out, "out", dev, dt, R, nq, hd)
    _apart(out, "out")
    pk, pv = _pool(k_pages, "k_pages", dev, dt, nkv, hd), _pool(v_pages, "v_pages", dev, dt, nkv, hd)
    if v_pages.shape != k_pages.shape:
        raise ValueError("k_pages and v_pages must have the same shape.")
    if nq == 0 or nkv == 0 or nq % nkv:
        raise ValueError("the query heads must be a positive multiple of the kv heads.")
    prefix_len = int(prefix_len)
    P = k_pages.shape[1]
    ppt = _vec(prefix_table, "prefix_table", dev, _I32) if prefix_table is not None else 0
    if prefix_len < 0 or (prefix_len and (not ppt or prefix_table.shape[0] * P < prefix_len)):
        raise ValueError("prefix_table does not hold prefix_len tokens.")
    if not isinstance(tables, torch.Tensor) or tables.device != dev or tables.dtype != _I32 or tables.dim() != 2 or \
            _gaps(tables):
        raise ValueError(f"tables must be int32 [requests, width] on {dev} with contiguous rows.")
    B, W = tables.shape
    pl = _vec(row_lens, "row_lens", dev, _I32, R)
    prs = 0
    if row_seq is not None:
        prs = _vec(row_seq, "row_seq", dev, _I32, R)
    elif B < R:
        raise ValueError("without row_seq the tables need a row for each row.")
    if R == 0:
        return
    scale = hd ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite.")
    # the stride of a dimension of one entry says nothing
    ks, vs = (tuple(st if n > 1 else hd for n, st in zip(t.shape, t.stride())) for t in (k_pages, v_pages))
    rest = (q.stride(0), q.stride(1), out.stride(0), out.stride(1), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], tables.stride(0),
            R, nq, nkv, hd, P, k_pages.shape[0], prefix_len, W, B, _DT[dt], scale, 0)
    L = lib()
    size = C.c_size_t()
    st = L.tt_shared_prefix_attention_workspace(_PREFIX.pack(pq, pk, pv, po, ppt, tables.data_ptr(), pl, prs, 0, *rest),
                                                C.byref(size))
    if st:
        check(st, "shared_prefix_attention")
    ws = torch.empty(size.value, dtype=torch.uint8, device=dev) if size.value else None
    _run(L.tt_shared_prefix_attention, _PREFIX.pack(pq, pk, pv, po, ppt, tables.data_ptr(), pl, prs,
                                                    0 if ws is None else ws.data_ptr(), *rest), dev, "shared_prefix_attention")
