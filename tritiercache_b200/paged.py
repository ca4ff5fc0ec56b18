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
import functools
import math
import struct
import threading

import torch

from ._lib import check, lib

_F32, _BF16, _F16, _I32, _I64 = torch.float32, torch.bfloat16, torch.float16, torch.int32, torch.int64
_DT = {_F32: 0, _BF16: 1, _F16: 2}

# the argument structs of the C ABI, packed with native alignment
_TABLES = struct.Struct("@14Pq6i")
_ROPE = struct.Struct("@12P18q12ifi")
_PREFIX = struct.Struct("@9P11q10ifi")

# torch.cuda.current_stream() builds a Stream object, at half the price of a whole call here
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)
_local = threading.local()


def _vec(t, name: str, index: int, dtype, n: int) -> int:
    """Address of a contiguous 1-D tensor of n elements."""
    if t.dtype is not dtype or t.shape != (n,) or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape [{n}] on cuda:{index}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}.")
    return t.data_ptr()


def _rows(t, name: str, index: int, dtype, shape):
    """Strides of a tensor of this shape whose last dimension has no gaps."""
    st = t.stride()
    if t.dtype is not dtype or t.shape != shape or t.get_device() != index or \
            (st[-1] != 1 and shape[-1] > 1 and t.numel() > 0):
        raise ValueError(f"{name} must be {dtype} {tuple(shape)} on cuda:{index} without gaps in its last dimension, got {t.dtype} "
                         f"{tuple(t.shape)}, strides {tuple(st)}, on {t.device}.")
    return st


def _apart(t, st, name: str) -> None:
    """An output whose dimensions overlap (an expanded one) would be written by several threads."""
    if 0 in st and any(d == 0 and n > 1 for n, d in zip(t.shape, st)):
        raise ValueError(f"{name} is an output and must not be an expanded tensor.")


def _device(t, name: str) -> int:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path).")
    return t.get_device()


def _run(fn, packed: bytes, index: int, what: str) -> None:
    if torch.cuda.current_device() == index:
        st = fn(packed, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            st = fn(packed, _raw_stream(index))
    if st:
        check(st, what)


def _tensors_only(fn):
    """What is not a tensor has none of a tensor's attributes; what is no 32-bit whole number does not pack, nor does a
    whole number that no float holds."""
    @functools.wraps(fn)
    def call(*args, **kw):
        try:
            return fn(*args, **kw)
        except AttributeError as e:
            raise ValueError(f"{fn.__name__} takes tensors: {e}") from None
        except (struct.error, OverflowError) as e:
            raise ValueError(f"{fn.__name__}: a number does not fit its type: {e}") from None
    return call


@_tensors_only
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
    index = _device(tables, "tables")
    if tables.dim() != 2:
        raise ValueError("tables must be int32 [requests, width].")
    B, W = tables.shape
    ts = _rows(tables, "tables", index, _I32, tables.shape)
    if B > 1 and ts[0] < W:
        raise ValueError("tables is written and its rows must not overlap.")
    n = slots.numel()
    cap = free_pages.numel()
    fc = _vec(free_count, "free_count", index, _I32, 1)
    L = lib()
    size = L.tt_page_tables_workspace(B, n)
    ws = torch.empty(size, dtype=torch.uint8, device=tables.device) if size else None
    packed = _TABLES.pack(_vec(ctx_lens, "ctx_lens", index, _I32, B), _vec(new_lens, "new_lens", index, _I32, B), tables.data_ptr(),
                          _vec(free_pages, "free_pages", index, _I32, cap), fc,
                          fc if free_count_out is None else _vec(free_count_out, "free_count_out", index, _I32, 1),
                          _vec(seq_lens, "seq_lens", index, _I32, B), _vec(cu_new, "cu_new", index, _I32, B + 1),
                          _vec(slots, "slots", index, _I64, n), _vec(positions, "positions", index, _I32, n),
                          _vec(row_seq, "row_seq", index, _I32, n), _vec(row_lens, "row_lens", index, _I32, n),
                          _vec(deferred, "deferred", index, _I32, 1), ws.data_ptr() if size else 0, ts[0] if B > 1 else W, B, W, cap,
                          page_size, n, position_offset)
    _run(L.tt_page_tables, packed, index, "page_tables")


@_tensors_only
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
    index = _device(q, "q")
    dt = q.dtype
    if dt not in _DT or q.dim() != 3 or k.dim() != 3:
        raise ValueError("q and k must be float32, bfloat16 or float16 [rows, heads, head_dim].")
    R, nq, hd = shape = q.shape
    nkv = k.shape[1]
    kv_shape = (R, nkv, hd)
    qt, kt = q_out.dtype, k_dst.dtype
    if (qt is not dt and qt is not _F32) or (kt is not dt and kt is not _F32):
        raise ValueError(f"q_out, k_dst and v_dst must be {dt} or float32.")
    if (v is None) != (v_dst is None):
        raise ValueError("v and v_dst come together.")
    qs, os = _rows(q, "q", index, dt, shape), _rows(q_out, "q_out", index, qt, shape)
    ks = _rows(k, "k", index, dt, kv_shape)
    if slots is None:
        dst, psl, pages, psize = kv_shape, 0, R, 1
    else:
        if k_dst.dim() != 4:
            raise ValueError("with slots k_dst and v_dst must be [pages, page_size, kv_heads, head_dim].")
        pages, psize = k_dst.shape[:2]
        dst, psl = (pages, psize, nkv, hd), _vec(slots, "slots", index, _I64, R)
    kd = _rows(k_dst, "k_dst", index, kt, dst)
    _apart(q_out, os, "q_out")
    _apart(k_dst, kd, "k_dst")
    vs, vd, pv, pvd = (0, 0), kd, 0, 0
    if v is not None:
        vs, vd = _rows(v, "v", index, dt, kv_shape), _rows(v_dst, "v_dst", index, kt, dst)
        _apart(v_dst, vd, "v_dst")
        pv, pvd = v.data_ptr(), v_dst.data_ptr()
    if slots is None:
        kd, vd = (kd[0], 0, kd[1]), (vd[0], 0, vd[1])
    wt, pqw, pkw = dt, 0, 0
    if q_weight is not None:
        wt = q_weight.dtype
        pqw = _vec(q_weight, "q_weight", index, wt, hd)
    if k_weight is not None:
        if q_weight is None:
            wt = k_weight.dtype
        pkw = _vec(k_weight, "k_weight", index, wt, hd)  # of one type with q_weight
    tt, pc, psn, cst, sst, trows, rot = dt, 0, 0, 0, 0, 0, 0
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together.")
    if cos is not None:
        tt = cos.dtype
        trows, half = cos.shape
        cst, sst = _rows(cos, "cos", index, tt, cos.shape)[0], _rows(sin, "sin", index, tt, cos.shape)[0]
        rot = 2 * half
        if rot:
            pc, psn = cos.data_ptr(), sin.data_ptr()
    if (wt is not dt and wt is not _F32) or (tt is not dt and tt is not _F32):
        raise ValueError(f"weights and tables must be {dt} or float32.")
    ppos, p64 = 0, 0
    if positions is not None:
        p64 = 1 if positions.dtype is _I64 else 0
        ppos = _vec(positions, "positions", index, _I64 if p64 else _I32, R)
    if R == 0:
        return
    packed = _ROPE.pack(q.data_ptr(), k.data_ptr(), pv, q_out.data_ptr(), k_dst.data_ptr(), pvd, pqw, pkw, pc, psn, ppos, psl,
                        qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os[0], os[1], kd[0], kd[1], kd[2], vd[0], vd[1], vd[2], cst, sst,
                        trows, pages, R, nq, nkv, hd, rot, psize, _DT[dt], _DT[qt], _DT[kt], _DT[wt], _DT[tt], p64, eps, 0)
    _run(lib().tt_qk_norm_rope, packed, index, "qk_norm_rope")


@_tensors_only
def shared_prefix_attention(q, k_pages, v_pages, prefix_table, prefix_len, tables, row_lens, out, row_seq=None,
                            scale=None) -> None:
    """Decode attention of a batch over a prefix that all rows share, read once
    for all of them, and over each row's own pages.

    ``q``, ``out`` [rows, q_heads, head_dim], channels contiguous, strides and
    start of q multiples of 2 elements; ``k_pages``/``v_pages`` [pages, page_size,
    kv_heads, head_dim], channels contiguous, other strides and start in 16-byte
    steps, page_size a power of two from 16; bfloat16 or float16 throughout.  Row r attends tokens
    [0, prefix_len) of the pages in ``prefix_table`` and tokens [0, row_lens[r])
    of the pages in row ``row_seq[r]`` (None: r) of ``tables``.  ``scale``
    defaults to head_dim ** -0.5.  Rows with row_seq < 0 are padding and stay as
    they were; a row with nothing to attend gives zeros; a page outside the pool
    or a length beyond the table gives NaN.  out may be q itself.
    """
    index = _device(q, "q")
    dt = q.dtype
    if (dt is not _BF16 and dt is not _F16) or q.dim() != 3:
        raise ValueError("q must be bfloat16 or float16 [rows, heads, head_dim].")
    R, nq, hd = shape = q.shape
    if k_pages.dim() != 4 or k_pages.shape[3] != hd:
        raise ValueError(f"k_pages must be [pages, page_size, kv_heads, {hd}].")
    pages, P, nkv, _ = pool = k_pages.shape
    if nq == 0 or nkv == 0 or nq % nkv:
        raise ValueError("the query heads must be a positive multiple of the kv heads.")
    qs, os = _rows(q, "q", index, dt, shape), _rows(out, "out", index, dt, shape)
    _apart(out, os, "out")
    ks, vs = _rows(k_pages, "k_pages", index, dt, pool), _rows(v_pages, "v_pages", index, dt, pool)
    if R == 1 or nq == 1:  # the stride of a dimension of one entry says nothing
        qs = tuple(d if n > 1 else hd for n, d in zip(shape, qs))
    if 1 in pool:
        ks, vs = (tuple(d if n > 1 else hd for n, d in zip(pool, st)) for st in (ks, vs))
    ppt, have = 0, 0
    if prefix_table is not None:
        have = prefix_table.numel()
        ppt = _vec(prefix_table, "prefix_table", index, _I32, have)
    if prefix_len < 0 or have * P < prefix_len:
        raise ValueError("prefix_table does not hold prefix_len tokens.")
    if tables.dim() != 2:
        raise ValueError("tables must be int32 [requests, width].")
    B, W = tables.shape
    ts = _rows(tables, "tables", index, _I32, tables.shape)
    pl = _vec(row_lens, "row_lens", index, _I32, R)
    prs = 0 if row_seq is None else _vec(row_seq, "row_seq", index, _I32, R)
    if row_seq is None and B < R:
        raise ValueError("without row_seq the tables need a row for each row.")
    if R == 0:
        return
    scale = hd ** -0.5 if scale is None else scale
    if not math.isfinite(scale):
        raise ValueError("scale must be finite.")
    first = (q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(), ppt, tables.data_ptr(), pl, prs)
    rest = (qs[0], qs[1], os[0], os[1], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], ts[0], R, nq, nkv, hd, P, pages, prefix_len, W, B,
            1 if dt is _BF16 else 2, scale, 0)
    L = lib()
    size = getattr(_local, "size", None)
    if size is None:
        size = _local.size = C.c_size_t()
    st = L.tt_shared_prefix_attention_workspace(_PREFIX.pack(*first, 0, *rest), C.byref(size))
    if st:
        check(st, "shared_prefix_attention")
    ws = torch.empty(size.value, dtype=torch.uint8, device=q.device) if size.value else None
    _run(L.tt_shared_prefix_attention, _PREFIX.pack(*first, 0 if ws is None else ws.data_ptr(), *rest), index,
         "shared_prefix_attention")


class SharedPrefixBatch:
    """A paged cache for requests that continue one shared prompt, and the
    calls of a step over it::

        batch = SharedPrefixBatch(num_pages, 16, num_kv_heads, head_dim, max_requests, max_pages, max_rows)
        slots, positions = batch.set_prefix(n)      # then qk_norm_rope of the prompt's rows into these slots
        batch.begin(new_lens)                       # pages, slots, positions of the step's rows
        batch.place(q, k, v, cos, sin, q_out)       # norm, rotation, keys and values into the pages
        batch.attend(q_out, out)                    # prompt once for all rows, then each row's own pages

    The buffers belong to the object and keep their addresses, so a step can be
    captured into a CUDA graph.  bfloat16 or float16, head_dim 64 or 128, pages of
    a power of two from 16 tokens.  No reference counterpart.  ``max_rows`` is the
    number of new tokens a step can hold; rows behind the step's are padding.
    After ``begin``: ``lens`` [requests] tokens held, ``row_seq`` [rows] the
    request of each row (-1: padding), ``deferred`` [1] the requests that found
    no pages and wait.
    """

    def __init__(self, num_pages, page_size, num_kv_heads, head_dim, max_requests, max_pages, max_rows,
                 dtype=torch.bfloat16, device=None):
        if min(num_pages, page_size, num_kv_heads, head_dim, max_requests, max_pages, max_rows) <= 0:
            raise ValueError("sizes must be positive.")
        # what attend() takes, said before the buffers are made
        if dtype is not _BF16 and dtype is not _F16:
            raise ValueError(f"dtype must be bfloat16 or float16, got {dtype}.")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {head_dim}.")
        if not 16 <= page_size <= 32768 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 32768, got {page_size}.")
        if max_pages * page_size > 2 ** 31 - 1:
            raise ValueError("max_pages * page_size must not exceed 2^31 - 1.")
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        shape = (num_pages, page_size, num_kv_heads, head_dim)
        self.k_pages, self.v_pages = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        new = lambda n, dt=_I32: torch.zeros(n, dtype=dt, device=device)  # noqa: E731
        self.tables = torch.full((max_requests, max_pages), -1, dtype=_I32, device=device)
        self.lens, self.cu_new, self.deferred = new(max_requests), new(max_requests + 1), new(1)
        self.slots, self.positions, self.row_seq, self.row_lens = new(max_rows, _I64), new(max_rows), new(max_rows), new(max_rows)
        self.free_pages = torch.arange(num_pages - 1, -1, -1, dtype=_I32, device=device)
        self.free_count = torch.full((1,), num_pages, dtype=_I32, device=device)
        self.page_size = page_size
        self.prefix_len = 0
        self.prefix_table = new(0)
        self._num_pages, self._begun = num_pages, False

    def set_prefix(self, length: int):
        """Gives the shared prompt its pages (before the first step); returns the
        slots and positions of its tokens."""
        pages = -(-length // self.page_size)
        if self._begun:
            raise ValueError("the prefix is set before the first step.")
        if length < 0 or pages > self._num_pages:
            raise ValueError("the pool does not hold the prefix.")
        dev = self.tables.device
        self.prefix_len = length
        self.prefix_table = torch.arange(pages, dtype=_I32, device=dev)  # the bottom of the stack is handed out last
        self.free_pages.copy_(torch.arange(self._num_pages - 1, -1, -1, dtype=_I32, device=dev))
        self.free_count.fill_(self._num_pages - pages)
        t = torch.arange(length, device=dev)
        return t, t.to(_I32)

    def begin(self, new_lens) -> None:
        """new_lens [requests] int32: new tokens, 0 rests, -1 has ended."""
        page_tables(self.lens, new_lens, self.tables, self.free_pages, self.free_count, self.page_size, self.lens, self.cu_new,
                    self.slots, self.positions, self.row_seq, self.row_lens, self.deferred, position_offset=self.prefix_len)
        self._begun = True

    def place(self, q, k, v, cos, sin, q_out, q_weight=None, k_weight=None, eps=1e-6) -> None:
        """qk_norm_rope of the step's rows ([max_rows, heads, head_dim]) into the pages."""
        qk_norm_rope(q, k, v, cos, sin, q_out, self.k_pages, self.v_pages, q_weight, k_weight, eps, self.positions, self.slots)

    def attend(self, q, out, scale=None) -> None:
        """shared_prefix_attention of the step's rows."""
        shared_prefix_attention(q, self.k_pages, self.v_pages, self.prefix_table, self.prefix_len, self.tables, self.row_lens, out,
                                row_seq=self.row_seq, scale=scale)
