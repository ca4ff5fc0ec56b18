"""Page tables, query/key norms with rotation, and shared-prefix attention on the GPU against plain
restatements (whole numbers exactly, computed numbers in 64 bits).

Tolerances count the roundings: u = finfo.eps / 2 of the output's type for the last one, the same again for
the attention weights (rounded to the pages' type before the second product), and float32 sums.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def C_():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from tritiercache_b200 import _C
    return _C


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def unit(dt):
    return torch.finfo(dt).eps / 2


# ---------------------------------------------------------------------------------------------
# page tables
# ---------------------------------------------------------------------------------------------
def tables_ref(ctx, new, tables, free, count, P, rows, offset):
    """The definition, request after request."""
    ctx = np.maximum(ctx, 0).astype(np.int64)
    tables, free = tables.copy(), free.copy()
    B, W = tables.shape
    cap = len(free)
    count = min(max(int(count), 0), cap)
    for b in range(B):
        if new[b] < 0:
            for j in range(min(-(-ctx[b] // P), W)):
                if count + j < cap:
                    free[count + j] = tables[b, j]
            count += min(-(-ctx[b] // P), W)
    count = min(count, cap)
    top, asked = count, 0
    seq = np.zeros(B, np.int64)
    cu = np.zeros(B + 1, np.int64)
    out = {k: np.full(rows, v, d) for k, v, d in (("slots", -1, np.int64), ("positions", 0, np.int32),
                                                  ("row_seq", -1, np.int32), ("row_lens", 0, np.int32))}
    late = 0
    given = 0
    for b in range(B):
        n = max(int(new[b]), 0)
        cu[b + 1] = cu[b] + n
        held, last = -(-ctx[b] // P), -(-(ctx[b] + n) // P)
        seq[b] = 0 if new[b] < 0 else ctx[b] + n
        if n == 0:
            continue
        if last > W or cu[b + 1] > rows:
            late += 1
            seq[b] = ctx[b]
            continue
        need = last - held
        if need and asked + need > top:
            asked += need
            late += 1
            seq[b] = ctx[b]
            continue
        for j in range(need):
            tables[b, held + j] = free[top - 1 - asked - j]
        asked += need
        given += need
        for i in range(n):
            pos = ctx[b] + i
            t = cu[b] + i
            out["slots"][t] = tables[b, pos // P] * P + pos % P
            out["positions"][t] = pos + offset
            out["row_seq"][t] = b
            out["row_lens"][t] = pos + 1
    return dict(tables=tables, free_pages=free, free_count=np.array([top - given]), seq_lens=seq,
                cu_new=np.minimum(cu, 2 ** 31 - 1),
                deferred=np.array([late]), **out)


def tables_case(seed, B, W, P, new_max, ctx_max, ended, free_share, rows=None):
    r = np.random.default_rng(seed)
    ctx = r.integers(0, ctx_max + 1, B).astype(np.int32)
    new = r.integers(0, new_max + 1, B).astype(np.int32)
    new[r.random(B) < ended] = -1
    held = np.minimum(-(-ctx // P), W)
    need = int(np.maximum(-(-(ctx + np.maximum(new, 0)) // P) - held, 0).sum())
    free_n = int(need * free_share)
    ids = r.permutation(int(held.sum()) + free_n + 8).astype(np.int32)
    tables = np.full((B, W), -1, np.int32)
    at = 0
    for b in range(B):
        tables[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
    free = np.full(int(held.sum()) + free_n + 8, -7, np.int32)
    free[:free_n] = ids[at:at + free_n]
    rows = int(np.maximum(new, 0).sum()) + 5 if rows is None else rows
    return ctx, new, tables, free, free_n, rows


def tables_gpu(C_, ctx, new, tables, free, count, P, rows, offset, in_place=False):
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    B = len(ctx)
    t = {"tables": d(tables), "free_pages": d(free), "free_count": d(np.array([count], np.int32))}
    i32 = lambda n: torch.full((n,), 99, device="cuda", dtype=torch.int32)  # noqa: E731
    c = d(ctx)
    t.update(seq_lens=c if in_place else i32(B), cu_new=i32(B + 1), slots=torch.full((rows,), 99, device="cuda"),
             positions=i32(rows), row_seq=i32(rows), row_lens=i32(rows), deferred=i32(1))
    fc = t["free_count"] if in_place else i32(1)
    C_.page_tables(c, d(new), t["tables"], t["free_pages"], t["free_count"], P, t["seq_lens"], t["cu_new"], t["slots"],
                   t["positions"], t["row_seq"], t["row_lens"], t["deferred"], free_count_out=None if in_place else fc,
                   position_offset=offset)
    t["free_count"] = fc
    return {k: v.cpu().numpy() for k, v in t.items()}


def same(got, want):
    for k, v in want.items():
        assert np.array_equal(got[k].astype(np.int64), v.astype(np.int64)), (k, got[k], v)


@pytest.mark.parametrize("B,W,P,new_max,ctx_max,ended,share", [
    (1, 4, 16, 1, 40, 0.0, 1.0),
    (3, 1, 16, 16, 0, 0.0, 1.0),       # empty requests, full pages
    (37, 9, 16, 1, 140, 0.3, 1.0),     # decode, some ended
    (64, 12, 1, 3, 9, 0.2, 0.5),       # pages of one token, too few of them
    (300, 20, 7, 50, 90, 0.1, 0.6),    # page size no power of two, deferred requests
    (300, 4, 16, 50, 60, 0.1, 1.0),    # tables too narrow for some
    (1500, 8, 32, 1, 250, 0.5, 0.0),   # nothing free but what ended requests give back
    (2049, 6, 16, 3, 64, 0.1, 0.8),    # two launches because of the requests
    (40, 80, 16, 900, 300, 0.1, 1.0),  # two launches because of the rows
    (5000, 10, 32, 20, 200, 0.2, 0.7),
])
def test_page_tables_match_the_definition(C_, B, W, P, new_max, ctx_max, ended, share):
    for seed in range(3):
        case = tables_case(seed, B, W, P, new_max, ctx_max, ended, share)
        ctx, new, tables, free, count, rows = case
        want = tables_ref(ctx, new, tables, free, count, P, rows, 11)
        same(tables_gpu(C_, ctx, new, tables, free, count, P, rows, 11), want)
        same(tables_gpu(C_, ctx, new, tables, free, count, P, rows, 11, in_place=True), want)


def test_page_tables_small_row_buffer_and_odd_values(C_):
    ctx, new, tables, free, count, rows = tables_case(5, 50, 9, 16, 30, 90, 0.1, 1.0)
    for cut in (0, 1, 17, rows // 2):
        want = tables_ref(ctx, new, tables, free, count, 16, cut, 0)
        same(tables_gpu(C_, ctx, new, tables, free, count, 16, cut, 0), want)
    ctx[3], new[4], new[5] = -8, -3, 2 ** 31 - 1  # counts as 0, ended, fits nowhere
    for c in (-5, 0, len(free), len(free) + 40):  # a height outside the stack is clamped
        want = tables_ref(ctx, new, tables, free, c, 16, rows, 0)
        same(tables_gpu(C_, ctx, new, tables, free, c, 16, rows, 0), want)


def test_page_tables_without_requests_pads_the_rows(C_):
    for rows in (0, 5, 9000):
        ctx = np.zeros(0, np.int32)
        tables = np.zeros((0, 4), np.int32)
        free = np.arange(6, dtype=np.int32)
        same(tables_gpu(C_, ctx, ctx, tables, free, 4, 16, rows, 0), tables_ref(ctx, ctx, tables, free, 4, 16, rows, 0))


def test_page_tables_strided_table_rows(C_):
    ctx, new, tables, free, count, rows = tables_case(9, 20, 6, 16, 10, 80, 0.1, 1.0)
    want = tables_ref(ctx, new, tables, free, count, 16, rows, 0)
    wide = torch.full((20, 11), 123, device="cuda", dtype=torch.int32)
    wide[:, :6] = torch.from_numpy(tables).cuda()
    i32 = lambda n: torch.zeros(n, device="cuda", dtype=torch.int32)  # noqa: E731
    C_.page_tables(torch.from_numpy(ctx).cuda(), torch.from_numpy(new).cuda(), wide[:, :6], torch.from_numpy(free).cuda(),
                   torch.tensor([count], device="cuda", dtype=torch.int32), 16, i32(20), i32(21),
                   torch.zeros(rows, device="cuda", dtype=torch.int64), i32(rows), i32(rows), i32(rows), i32(1))
    assert np.array_equal(wide[:, :6].cpu().numpy(), want["tables"])
    assert bool((wide[:, 6:] == 123).all())


# ---------------------------------------------------------------------------------------------
# norm, rotation, placing
# ---------------------------------------------------------------------------------------------
def rope_ref(x, w, eps, cos, sin, rot):
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    h = rot // 2
    if h:
        c, s = cos.double()[:, None], sin.double()[:, None]
        a, b = x[..., :h], x[..., h:rot]
        x = torch.cat([a * c - b * s, b * c + a * s, x[..., rot:]], -1)
    return x


def rope_close(got, want, src, w, dt, hd):
    """One rounding to the output's type, and float32 steps: the sum of hd squares (hd + 3 roundings under the
    root, halved by it), scaling, weight and two products and a sum of the rotation, on either channel of a pair."""
    size = want.abs().amax(-1, keepdim=True)
    lim = unit(dt) * want.abs() + (hd / 2 + 8) * 2.0 ** -24 * 2 * size + (2.0 ** -25 if dt == F16 else 0)
    err = (got.double() - want).abs()
    assert bool((err <= lim).all()), float((err - lim).max())


@pytest.mark.parametrize("T,nq,nkv,hd,rot,norm,dt,odt,paged", [
    (1, 32, 8, 128, 128, True, BF, F32, False),
    (1, 4, 1, 64, 64, True, F16, F16, True),
    (3, 28, 4, 128, 128, False, BF, BF, True),
    (130, 12, 3, 64, 32, True, F16, F16, True),     # half of the head rotated
    (77, 6, 2, 256, 256, True, BF, BF, False),
    (50, 3, 3, 96, 96, True, BF, F32, True),        # 6 of 8 lanes at work
    (9, 5, 5, 80, 40, True, F32, F32, False),       # a rotation that 16-byte loads do not fit
    (9, 2, 1, 80, 20, True, BF, BF, True),
    (33, 4, 2, 2, 2, True, F32, F32, False),        # the smallest head
    (11, 2, 1, 512, 512, True, F32, F32, True),     # the largest
    (11, 2, 1, 512, 128, True, F16, F32, False),
    (5, 2, 1, 510, 34, True, BF, BF, False),
    (40, 8, 2, 128, 0, True, F16, F16, False),      # no rotation
    (2500, 32, 8, 128, 128, True, BF, BF, True),
    (4000, 4, 2, 64, 64, False, F32, F32, True),
])
def test_norm_rope_matches_the_formula(C_, T, nq, nkv, hd, rot, norm, dt, odt, paged):
    g = gen(T + hd)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    qkv = r(T, (nq + 2 * nkv) * hd).to(dt)
    q, k, v = (x.view(T, -1, hd) for x in qkv.split([nq * hd, nkv * hd, nkv * hd], 1))
    before = qkv.clone()
    q[0, 0].zero_()  # a head of zeros: eps keeps it finite
    before = qkv.clone()
    wq, wk = (1 + 0.3 * r(hd)).to(dt), (1 + 0.3 * r(hd)).to(dt)
    most = 3 * T + 7
    cos = sin = None
    pos = torch.randperm(most, generator=g, device="cuda")[:T].to(torch.int32)
    if rot:
        ang = r(most, rot // 2) * 50
        cos, sin = ang.cos(), ang.sin()
    q_out = torch.full((T, nq, hd), 7.0, device="cuda", dtype=odt)
    P = 16
    if paged:
        n = T // P + 3
        kd, vd = (torch.full((n, P, nkv, hd), 7.0, device="cuda", dtype=odt) for _ in range(2))
        slots = torch.randperm(n * P, generator=g, device="cuda")[:T]
        slots[T // 2::9] = -1
        if T > 20:
            slots[3] = n * P  # outside the pool: padding too
    else:
        kd, vd = (torch.full((T, nkv, hd), 7.0, device="cuda", dtype=odt) for _ in range(2))
        slots = None
    C_.qk_norm_rope(q, k, v, cos, sin, q_out, kd, vd, wq if norm else None, wk if norm else None, 1e-5, pos, slots)
    assert torch.equal(qkv, before)
    p = pos.long()
    c, s = (cos[p], sin[p]) if rot else (None, None)
    qr = rope_ref(q, wq if norm else None, 1e-5, c, s, rot)
    kr = rope_ref(k, wk if norm else None, 1e-5, c, s, rot)
    if paged:
        live = (slots >= 0) & (slots < n * P)
        rope_close(q_out[live], qr[live], q, wq, odt, hd)
        assert bool((q_out[~live] == 7).all())
        rope_close(kd.view(-1, nkv, hd)[slots[live]], kr[live], k, wk, odt, hd)
        assert torch.equal(vd.view(-1, nkv, hd)[slots[live]], v[live].to(odt))
        rest = torch.ones(n * P, dtype=torch.bool, device="cuda")
        rest[slots[live]] = False
        assert bool((kd.view(-1, nkv, hd)[rest] == 7).all()) and bool((vd.view(-1, nkv, hd)[rest] == 7).all())
    else:
        rope_close(q_out, qr, q, wq, odt, hd)
        rope_close(kd, kr, k, wk, odt, hd)
        assert torch.equal(vd, v.to(odt))


def test_norm_rope_in_place_low_tables_and_bad_positions(C_):
    g = gen(3)
    T, nq, nkv, hd = 19, 8, 2, 128
    q = torch.randn((T, nq, hd), generator=g, device="cuda").to(BF)
    k, v = (torch.randn((T, nkv, hd), generator=g, device="cuda").to(BF) for _ in range(2))
    ang = torch.randn((64, hd // 2), generator=g, device="cuda") * 9
    cos, sin = ang.cos().to(BF), ang.sin().to(BF)
    full = torch.cat([cos, cos], 1)  # both halves, as models keep them: a strided view is taken
    pos = torch.randint(0, 64, (T,), generator=g, device="cuda")  # int64
    pos[4], pos[9] = -1, 64
    w = 1 + 0.1 * torch.randn(hd, generator=g, device="cuda")
    want_q = rope_ref(q, w, 1e-6, cos[pos.clamp(0, 63)], sin[pos.clamp(0, 63)], hd)
    want_k = rope_ref(k, None, 1e-6, cos[pos.clamp(0, 63)], sin[pos.clamp(0, 63)], hd)
    v0 = v.clone()
    C_.qk_norm_rope(q, k, v, full[:, :hd // 2], sin, q, k, v, q_weight=w, positions=pos)
    ok = torch.ones(T, dtype=torch.bool, device="cuda")
    ok[4] = ok[9] = False
    rope_close(q[ok], want_q[ok], q, w, BF, hd)
    rope_close(k[ok], want_k[ok], k, None, BF, hd)
    assert bool(torch.isnan(q[~ok]).all()) and bool(torch.isnan(k[~ok]).all())
    assert torch.equal(v, v0)


def test_norm_rope_without_values_and_positions(C_):
    g = gen(4)
    q = torch.randn((5, 4, 64), generator=g, device="cuda")
    k = torch.randn((5, 2, 64), generator=g, device="cuda")
    ang = torch.randn((5, 32), generator=g, device="cuda")
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    C_.qk_norm_rope(q, k, None, ang.cos(), ang.sin(), qo, ko, None)
    rope_close(qo, rope_ref(q, None, 0, ang.cos(), ang.sin(), 64), q, None, F32, 64)
    rope_close(ko, rope_ref(k, None, 0, ang.cos(), ang.sin(), 64), k, None, F32, 64)


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
def make_attn(seed, R, nq, nkv, hd, prefix, lens, P, dt, chunk=1, layout="nhd", spare=3):
    g = gen(seed)
    lens = np.asarray(lens, np.int32)
    assert len(lens) == R
    seqs = -(-R // chunk)
    most = np.array([lens[s * chunk:(s + 1) * chunk].max() for s in range(seqs)])
    need = -(-most // P)
    W = max(1, int(need.max()) + 1)
    npre = -(-prefix // P)
    pages = npre + int(need.sum()) + spare
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    tables = torch.full((seqs, W), -1, device="cuda", dtype=torch.int32)
    at = npre
    for s in range(seqs):
        tables[s, :need[s]] = order[at:at + need[s]]
        at += int(need[s])
    shape = {"nhd": (pages, P, nkv, hd), "hnd": (pages, nkv, P, hd), "kv": (pages, 2, P, nkv, hd)}[layout]
    if layout == "kv":
        kv = torch.randn(shape, generator=g, device="cuda").to(dt)
        k, v = kv[:, 0], kv[:, 1]
    else:
        k, v = (torch.randn(shape, generator=g, device="cuda").to(dt) for _ in range(2))
        if layout == "hnd":
            k, v = k.permute(0, 2, 1, 3), v.permute(0, 2, 1, 3)
    q = torch.randn((R, nq, hd), generator=g, device="cuda").to(dt) * 2
    seq = torch.arange(R, device="cuda", dtype=torch.int32) // chunk
    return dict(q=q, k=k, v=v, ptab=order[:npre].contiguous(), prefix=prefix, tables=tables,
                lens=torch.from_numpy(lens).cuda(), seq=seq, P=P)


def poison_tail(s):
    """NaN and infinities in every place behind a length: the rest of the last pages, and the pages no one holds."""
    P = s["P"]
    pages = s["k"].shape[0]
    used = torch.zeros(pages * P, dtype=torch.bool, device="cuda")
    t = torch.arange(s["prefix"], device="cuda")
    used[s["ptab"].long()[t // P] * P + t % P] = True
    for r in range(len(s["lens"])):
        t = torch.arange(int(s["lens"][r]), device="cuda")
        used[s["tables"][int(s["seq"][r])].long()[t // P] * P + t % P] = True
    bad = ~used.view(pages, P)
    for x in (s["k"], s["v"]):
        x[bad] = float("nan")
    s["v"][bad & (torch.arange(P, device="cuda") % 2 == 0)[None]] = float("inf")


def attn_ref(s, scale):
    """(out, sum of weights times |v|, key count, largest |q||k| scale) in 64 bits."""
    P = s["P"]
    R, nq, hd = s["q"].shape
    nkv = s["k"].shape[2]
    out = torch.zeros((R, nq, hd), dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    reach = 0.0
    t = torch.arange(s["prefix"], device="cuda")
    pg = s["ptab"].long()
    kp, vp = (x[pg[t // P], t % P].double() for x in (s["k"], s["v"]))
    for r in range(R):
        t = torch.arange(int(s["lens"][r]), device="cuda")
        pg = s["tables"][int(s["seq"][r])].long()
        k = torch.cat([kp, s["k"][pg[t // P], t % P].double()])
        v = torch.cat([vp, s["v"][pg[t // P], t % P].double()])
        if not len(k):
            continue
        q = s["q"][r].double().view(nkv, nq // nkv, hd)
        w = torch.softmax(torch.einsum("hgd,thd->hgt", q, k) * scale, -1)
        out[r] = torch.einsum("hgt,thd->hgd", w, v).reshape(nq, hd)
        mag[r] = torch.einsum("hgt,thd->hgd", w, v.abs()).reshape(nq, hd)
        reach = max(reach, float(q.norm(dim=-1).max() * k.norm(dim=-1).max()) * abs(scale))
    return out, mag, reach


def attn_close(got, s, scale):
    """|error| <= u |out| (last rounding) + u sum w|v| (weights rounded to the pages' type) + float32: logits of hd
    products summed in a tensor core (2^-23 of the largest product sum for each addition), twice because weight and
    sum both follow them, exponentials and sums (2^-20 in all); f16 weights below 2^-14 are off by 2^-25 of a sum that
    is at least 1."""
    want, mag, reach = attn_ref(s, scale)
    dt, hd = got.dtype, got.shape[-1]
    u = unit(dt)
    keys = s["prefix"] + int(s["lens"].max())
    lim = u * want.abs() + mag * (u + 2 * hd * 2.0 ** -23 * reach + 2.0 ** -20) * 1.01
    if dt == F16:
        lim = lim + keys * 2.0 ** -25 * 8 + 2.0 ** -25
    err = (got.double() - want).abs()
    assert bool((err <= lim).all()), (float((err - lim).max()), float(err.max()))


def attend(C_, s, scale=None, rows=True, out=None):
    out = torch.full_like(s["q"], 5.0) if out is None else out
    C_.shared_prefix_attention(s["q"], s["k"], s["v"], s["ptab"], s["prefix"], s["tables"], s["lens"], out,
                               row_seq=s["seq"] if rows else None, scale=scale)
    return out


CASES = [
    # R, nq, nkv, hd, prefix, longest own, page, type, rows a request, layout
    (1, 8, 2, 128, 0, 1, 16, BF, 1, "nhd"),          # one token
    (1, 28, 4, 128, 700, 333, 16, BF, 1, "nhd"),     # one row
    (2, 4, 4, 64, 1, 17, 16, F16, 1, "nhd"),
    (3, 8, 1, 128, 127, 40, 32, F16, 1, "hnd"),
    (5, 12, 1, 64, 128, 100, 64, BF, 1, "kv"),       # 12 query heads a kv head
    (4, 34, 2, 128, 129, 70, 16, F16, 1, "nhd"),     # 17: two tiles of heads
    (7, 14, 2, 128, 1000, 64, 128, BF, 1, "hnd"),
    (6, 32, 8, 128, 2049, 600, 256, BF, 3, "nhd"),   # several rows a request, pages larger than a tile
    (33, 8, 8, 64, 515, 90, 32, F16, 1, "kv"),       # MHA
    (40, 28, 4, 128, 3000, 50, 16, BF, 4, "nhd"),    # 280 rows of heads
    (130, 16, 2, 64, 1300, 33, 16, BF, 1, "nhd"),
    (64, 16, 2, 128, 4500, 20, 32, F16, 2, "nhd"),   # 512 rows of heads, spans that cross kv heads
]


@pytest.mark.parametrize("R,nq,nkv,hd,prefix,most,P,dt,chunk,layout", CASES)
def test_attention_matches_the_formula(C_, R, nq, nkv, hd, prefix, most, P, dt, chunk, layout):
    r = np.random.default_rng(R + prefix)
    lens = r.integers(0, most + 1, R)
    lens[0] = most
    if R > 3:
        lens[1], lens[2] = 0, 1
    s = make_attn(R + hd, R, nq, nkv, hd, prefix, lens, P, dt, chunk, layout)
    poison_tail(s)
    attn_close(attend(C_, s), s, hd ** -0.5)


def test_attention_with_large_logits_and_rising_maxima(C_):
    for dt in (BF, F16):
        s = make_attn(1, 9, 8, 2, 128, 900, np.arange(9) * 40, 16, dt)
        # the best key last in the prefix and last in the rows: every reference is raised
        ramp = torch.arange(1, s["k"].shape[0] + 1, device="cuda").to(dt) / 8
        s["k"] *= ramp[:, None, None, None]
        attn_close(attend(C_, s, scale=0.3), s, 0.3)
        attn_close(attend(C_, s, scale=-0.3), s, -0.3)
        attn_close(attend(C_, s, scale=0.0), s, 0.0)


def test_attention_empty_rows_padding_and_in_place(C_):
    s = make_attn(2, 6, 8, 2, 64, 0, [0, 5, 0, 40, 1, 16], 16, BF)
    s["seq"][3] = -1
    out = attend(C_, s)
    assert bool((out[0] == 0).all()) and bool((out[2] == 0).all())
    assert bool((out[3] == 5).all())
    live = [1, 4, 5]
    keep = {k: (v[live] if k in ("q", "lens", "seq") else v) for k, v in s.items()}
    attn_close(out[live], keep, 64 ** -0.5)
    want = attend(C_, s, out=s["q"].clone())
    attend(C_, s, out=s["q"])
    assert torch.equal(s["q"], want)


def test_attention_padding_does_not_hide_the_prefix(C_):
    s = make_attn(3, 20, 8, 2, 128, 777, np.full(20, 9), 16, F16)
    s["q"][5] = float("nan")  # a padded row's query may hold anything
    s["seq"][5] = -1
    out = attend(C_, s)
    live = [r for r in range(20) if r != 5]
    keep = {k: (v[live] if k in ("q", "lens", "seq") else v) for k, v in s.items()}
    attn_close(out[live], keep, 128 ** -0.5)
    assert bool((out[5] == 5).all())


def test_attention_bad_pages_and_lengths_give_nan(C_):
    for R in (4, 40):
        s = make_attn(4, R, 8, 2, 128, 300, np.full(R, 50), 16, BF)
        good = attend(C_, s)
        s["tables"][1, 2] = s["k"].shape[0]      # beyond the pool
        s["tables"][2, 0] = -3
        s["lens"][3] = s["tables"].shape[1] * 16 + 1
        out = attend(C_, s)
        assert bool(torch.isnan(out[1:4]).all())
        assert torch.equal(out[0], good[0]) and torch.equal(out[4:], good[4:])
        s["seq"][0] = s["tables"].shape[0]
        assert bool(torch.isnan(attend(C_, s)[0]).all())
        s["seq"][0] = 0
        s["ptab"][7] = 1 << 30
        assert bool(torch.isnan(attend(C_, s)).all())
        s["ptab"][7] = -1
        assert bool(torch.isnan(attend(C_, s)).all())


def test_attention_nan_and_infinity_in_keys_reach_their_rows_only(C_):
    s = make_attn(5, 20, 4, 2, 64, 200, np.full(20, 30), 16, BF)
    good = attend(C_, s)
    s["v"][s["tables"][3, 1].long(), 2, 0] = float("nan")  # token 18 of row 3, kv head 0
    s["k"][s["tables"][6, 0].long(), 0, 1] = float("nan")
    out = attend(C_, s)
    assert bool(torch.isnan(out[3, :2]).all()) and bool(torch.isnan(out[6, 2:]).all())
    assert torch.equal(out[3, 2:], good[3, 2:]) and torch.equal(out[6, :2], good[6, :2])
    rest = [r for r in range(20) if r not in (3, 6)]
    assert torch.equal(out[rest], good[rest])


def test_attention_repeats_bit_for_bit(C_):
    s = make_attn(6, 70, 32, 8, 128, 2500, np.arange(70) * 5, 32, BF)
    a = attend(C_, s)
    for _ in range(3):
        assert torch.equal(attend(C_, s), a)


def test_attention_strided_queries_and_outputs(C_):
    s = make_attn(7, 12, 8, 2, 128, 400, np.full(12, 33), 16, F16)
    wide = torch.zeros((12, 11, 130), device="cuda", dtype=F16)
    wide[:, 2:10, :128] = s["q"]
    ref = attend(C_, s)
    o = torch.full((12, 9, 131), 5.0, device="cuda", dtype=F16)
    C_.shared_prefix_attention(wide[:, 2:10, :128], s["k"], s["v"], s["ptab"], 400, s["tables"], s["lens"], o[:, 1:, 1:129])
    assert torch.equal(o[:, 1:, 1:129], ref)
    assert bool((o[:, 0] == 5).all()) and bool((o[:, :, 0] == 5).all()) and bool((o[:, :, 129:] == 5).all())


def test_attention_on_a_side_stream_and_in_a_graph(C_):
    s = make_attn(8, 24, 16, 4, 128, 1500, np.full(24, 60), 16, BF)
    ref = attend(C_, s)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    out = torch.zeros_like(s["q"])
    with torch.cuda.stream(st):
        attend(C_, s, out=out)
    st.synchronize()
    assert torch.equal(out, ref)
    outs = [torch.zeros_like(s["q"]) for _ in range(2)]
    graphs = []
    for o in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            attend(C_, s, out=o)
        graphs.append(g)
    # both graphs in flight at once: each has its own workspace
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(a):
            graphs[0].replay()
        with torch.cuda.stream(b):
            graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], ref) and torch.equal(outs[1], ref)
    # lengths change between replays without a new capture
    s["lens"].fill_(7)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], attend(C_, s))


# ---------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------
def test_serving_steps_together(C_):
    """Prompts in chunks, then single tokens, requests that end and pages that run short: every step's outputs
    against attention over the keys kept in a plain list."""
    g = gen(10)
    B, W, P, nq, nkv, hd, prefix = 9, 8, 16, 8, 2, 128, 150
    pool, rows = 21, 64  # eleven pages for nine requests: some wait
    k_pages, v_pages = (torch.full((pool, P, nkv, hd), float("nan"), device="cuda", dtype=BF) for _ in range(2))
    npre = -(-prefix // P)
    ptab = torch.arange(npre, device="cuda", dtype=torch.int32)
    ang = torch.arange(600, device="cuda")[:, None] * (1e4 ** (-torch.arange(0, hd, 2, device="cuda") / hd))[None]
    cos, sin = ang.cos(), ang.sin()
    w = (1 + 0.1 * torch.randn(hd, generator=g, device="cuda")).to(BF)
    i32 = lambda n, v=0: torch.full((n,), v, device="cuda", dtype=torch.int32)  # noqa: E731

    def place(T, positions, slots, q_out):
        qkv = torch.randn((T, (nq + 2 * nkv) * hd), generator=g, device="cuda").to(BF)
        q, k, v = (x.view(T, -1, hd) for x in qkv.split([nq * hd, nkv * hd, nkv * hd], 1))
        C_.qk_norm_rope(q, k, v, cos, sin, q_out, k_pages, v_pages, w, w, positions=positions, slots=slots)

    # the shared prompt itself, through the same call
    t = torch.arange(prefix, device="cuda")
    place(prefix, t.to(torch.int32), ptab.long()[t // P] * P + t % P, torch.empty((prefix, nq, hd), device="cuda", dtype=BF))
    lens, tables = i32(B), torch.full((B, W), -1, device="cuda", dtype=torch.int32)
    free = torch.arange(pool - 1, -1, -1, device="cuda", dtype=torch.int32)
    count = i32(1, pool - npre)
    slots = torch.zeros(rows, device="cuda", dtype=torch.int64)
    pos, seq, rl, cu, late = i32(rows), i32(rows), i32(rows), i32(B + 1), i32(1)
    r = np.random.default_rng(1)
    lates = 0
    for step in range(14):
        new = r.integers(1, 22, B) if step < 3 else np.ones(B, np.int64)
        new[r.random(B) < 0.15] = 0
        if step > 3:
            new[r.random(B) < 0.2] = -1
        while np.maximum(new, 0).sum() > rows:
            new[np.argmax(new)] //= 2
        h_lens = lens.cpu().numpy().copy()
        C_.page_tables(lens, torch.from_numpy(new.astype(np.int32)).cuda(), tables, free, count, P, lens, cu, slots, pos, seq, rl,
                       late, position_offset=prefix)
        lates += int(late)
        q = torch.full((rows, nq, hd), float("nan"), device="cuda", dtype=BF)
        out = torch.full((rows, nq, hd), 5.0, device="cuda", dtype=BF)
        place(rows, pos, slots, q)
        C_.shared_prefix_attention(q, k_pages, v_pages, ptab, prefix, tables, rl, out, row_seq=seq)
        live = (seq >= 0).nonzero().flatten()
        assert bool((out[seq < 0] == 5).all()) and bool(torch.isfinite(out).all())
        held = [p for b in range(B) if int(lens[b]) for p in tables[b, :-(-int(lens[b]) // P)].tolist()]
        stack = free[:int(count)].tolist()
        assert sorted(held + stack + ptab.tolist()) == list(range(pool))  # every page is in one place
        if len(live):
            s = dict(q=q[live], k=k_pages, v=v_pages, ptab=ptab, prefix=prefix, tables=tables, lens=rl[live], seq=seq[live], P=P)
            attn_close(out[live], s, hd ** -0.5)
        got = lens.cpu().numpy()
        assert all(got[b] in (0 if new[b] < 0 else h_lens[b] + max(new[b], 0), h_lens[b]) for b in range(B))
    assert lates > 0


def test_python_calls_refuse_what_does_not_fit(C_):
    s = make_attn(11, 3, 8, 2, 128, 40, [4, 5, 6], 16, BF)
    ok = dict(q=s["q"], k_pages=s["k"], v_pages=s["v"], prefix_table=s["ptab"], prefix_len=40, tables=s["tables"],
              row_lens=s["lens"], out=torch.empty_like(s["q"]))
    for bad in (dict(q=s["q"].float()), dict(q=s["q"][:, :7]), dict(q=s["q"].cpu()), dict(out=s["q"].half()), dict(prefix_len=49),
                dict(prefix_len=-1), dict(prefix_table=None), dict(prefix_table=s["ptab"].long()), dict(tables=s["tables"][:2]),
                dict(row_lens=s["lens"][:2]), dict(row_lens=s["lens"].long()), dict(v_pages=s["v"][:3]), dict(k_pages=s["k"].half()),
                dict(k_pages=s["k"][:, :8], v_pages=s["v"][:, :8]), dict(out=torch.empty_like(s["q"][:1]).expand(3, 8, 128)),
                dict(scale=float("nan")), dict(row_seq=s["lens"][:2]), dict(q=s["q"].transpose(1, 2))):
        with pytest.raises(ValueError):
            C_.shared_prefix_attention(**{**ok, **bad})
    q, k = torch.zeros((3, 4, 64), device="cuda"), torch.zeros((3, 2, 64), device="cuda")
    cos = torch.zeros((9, 32), device="cuda")
    ok = dict(q=q, k=k, v=k, cos=cos, sin=cos, q_out=q, k_dst=k, v_dst=k)
    for bad in (dict(q=q[0]), dict(k=k[:2]), dict(v=None), dict(sin=None), dict(sin=cos[:, :31]), dict(cos=cos.half(), sin=cos.half()),
                dict(q_out=q.half()), dict(k_dst=k[:, :1]), dict(q_weight=torch.zeros(63, device="cuda")),
                dict(q_weight=torch.zeros(64, device="cuda", dtype=BF)), dict(positions=torch.zeros(2, device="cuda", dtype=torch.int32)),
                dict(positions=torch.zeros(3, device="cuda")), dict(slots=torch.zeros(3, device="cuda", dtype=torch.int64)),
                dict(cos=cos[:2], sin=cos[:2]), dict(q_out=q[:1].expand(3, 4, 64)), dict(cos=torch.zeros((9, 33), device="cuda"),
                                                                                          sin=torch.zeros((9, 33), device="cuda"))):
        with pytest.raises(ValueError):
            C_.qk_norm_rope(**{**ok, **bad})
    i32 = lambda n: torch.zeros(n, device="cuda", dtype=torch.int32)  # noqa: E731
    ok = dict(ctx_lens=i32(2), new_lens=i32(2), tables=torch.zeros((2, 4), device="cuda", dtype=torch.int32), free_pages=i32(5),
              free_count=i32(1), page_size=16, seq_lens=i32(2), cu_new=i32(3), slots=i32(4).long(), positions=i32(4), row_seq=i32(4),
              row_lens=i32(4), deferred=i32(1))
    for bad in (dict(ctx_lens=i32(3)), dict(cu_new=i32(2)), dict(slots=i32(4)), dict(positions=i32(3)), dict(page_size=0),
                dict(tables=ok["tables"].t()), dict(free_count=i32(2)), dict(deferred=None), dict(new_lens=i32(2).cpu())):
        with pytest.raises(ValueError):
            C_.page_tables(**{**ok, **bad})
    torch.cuda.synchronize()


def test_numbers_that_do_not_fit_are_refused(C_):
    s = make_attn(12, 3, 8, 2, 128, 40, [4, 5, 6], 16, BF)
    i32 = lambda n: torch.zeros(n, device="cuda", dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError):
        C_.shared_prefix_attention(s["q"], s["k"], s["v"], s["ptab"], 2 ** 40, s["tables"], s["lens"], torch.empty_like(s["q"]))
    for kw in (dict(page_size=16.5), dict(page_size=2 ** 33), dict(position_offset=2 ** 31)):
        with pytest.raises(ValueError):
            C_.page_tables(i32(2), i32(2), torch.zeros((2, 4), device="cuda", dtype=torch.int32), i32(5), i32(1),
                           seq_lens=i32(2), cu_new=i32(3), slots=i32(4).long(), positions=i32(4), row_seq=i32(4), row_lens=i32(4),
                           deferred=i32(1), **{"page_size": 16, **kw})


def test_attention_of_pools_with_shared_heads_and_single_pages(C_):
    # the strides of dimensions of one entry say nothing, and heads may lie over one another (read only)
    s = make_attn(13, 5, 8, 1, 128, 30, [1, 2, 3, 4, 5], 32, BF)
    want = attend(C_, s)
    one = {**s, "k": s["k"].as_strided(s["k"].shape, (*s["k"].stride()[:2], 3, 1)),
           "v": s["v"].as_strided(s["v"].shape, (*s["v"].stride()[:2], 5, 1))}
    assert torch.equal(attend(C_, one), want)
    q = s["q"].repeat(1, 2, 1)
    four = {**s, "q": q, "k": s["k"].expand(-1, -1, 2, -1), "v": s["v"].expand(-1, -1, 2, -1)}
    got = attend(C_, four)
    assert torch.equal(got[:, :8], want) and torch.equal(got[:, 8:], want)


def test_attention_in_large_pools_and_pages(C_):
    """Offsets beyond 32 bits: the pages in use lie at the end of a pool of over 2^32 bytes and 2^31 elements."""
    P, nkv, hd, pages = 32768, 8, 128, 72
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 20 GB of device memory")
    k, v = (torch.empty((pages, P, nkv, hd), device="cuda", dtype=BF) for _ in range(2))
    assert k.numel() > 2 ** 31
    g = gen(14)
    for p in (70, 71):
        for x in (k, v):
            x[p] = torch.randn((P, nkv, hd), generator=g, device="cuda").to(BF)
    R = 6
    s = dict(q=torch.randn((R, 16, hd), generator=g, device="cuda").to(BF), k=k, v=v,
             ptab=torch.tensor([71], device="cuda", dtype=torch.int32), prefix=700,
             tables=torch.full((R, 1), 70, device="cuda", dtype=torch.int32),
             lens=torch.tensor([1, 40, 333, 1000, 7, 0], device="cuda", dtype=torch.int32),
             seq=torch.arange(R, device="cuda", dtype=torch.int32), P=P)
    attn_close(attend(C_, s), s, hd ** -0.5)
    slots = torch.tensor([71 * P + 5, 70 * P + 9], device="cuda")
    x = torch.randn((2, nkv, hd), generator=g, device="cuda").to(BF)
    q = torch.zeros((2, 16, hd), device="cuda", dtype=BF)
    C_.qk_norm_rope(q, x, x, None, None, q, k, v, slots=slots)
    assert torch.equal(k.view(-1, nkv, hd)[slots], x) and torch.equal(v.view(-1, nkv, hd)[slots], x)


def test_first_calls_may_be_captured(C_):
    """In a process of their own: the first call of each operator is inside a stream capture."""
    import subprocess
    import sys
    code = """
import sys; sys.path[:0] = ['.', 'tests']
import torch, test_gpu_paged as t
from tritiercache_b200 import _C
s = t.make_attn(1, 9, 8, 2, 128, 300, [3] * 9, 16, torch.bfloat16)
q = torch.zeros_like(s['q']); k = torch.zeros((9, 2, 128), device='cuda', dtype=torch.bfloat16)
out = torch.zeros_like(q)
i32 = lambda n: torch.zeros(n, device='cuda', dtype=torch.int32)
a = [i32(2), i32(2), torch.zeros((2, 4), device='cuda', dtype=torch.int32), i32(5), i32(1), 16, i32(2), i32(3), i32(9000).long(),
     i32(9000), i32(9000), i32(9000), i32(1)]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    _C.qk_norm_rope(q, k, k, None, None, q, k, k)
    _C.page_tables(*a)
    t.attend(_C, s, out=out)
g.replay()
torch.cuda.synchronize()
assert torch.equal(out, t.attend(_C, s)) and int(a[8][0]) == -1
print('captured')
"""
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=root, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


# ---------------------------------------------------------------------------------------------
# attention at sizes where the shared prefix has a pass of its own
# ---------------------------------------------------------------------------------------------
SHARED = [
    # R, nq, nkv, hd, prefix, longest own, page, type, rows a request, layout
    (70, 8, 8, 128, 127, 20, 16, BF, 1, "nhd"),      # one head a kv head, a prefix short of a tile
    (66, 16, 8, 128, 128, 20, 32, F16, 1, "hnd"),
    (65, 8, 8, 128, 129, 40, 16, BF, 1, "kv"),       # a tile of one key
    (300, 16, 2, 128, 130, 10, 64, F16, 3, "nhd"),   # 2400 rows of heads a kv head: ten row tiles
    (33, 24, 8, 128, 1000, 50, 128, BF, 1, "hnd"),   # 99 rows of heads: even and odd key tiles
    (16, 64, 8, 128, 1024, 30, 256, F16, 1, "nhd"),  # 128 rows of heads exactly
    (17, 64, 8, 128, 1025, 30, 32, BF, 1, "nhd"),    # 136: the second half almost empty
    (90, 6, 3, 64, 777, 60, 16, F16, 2, "kv"),
    (200, 12, 1, 64, 999, 30, 16, BF, 1, "nhd"),     # 12 heads: two tiles of 8 in the rows' pass
    (40, 34, 2, 128, 2000, 20, 16, BF, 1, "nhd"),    # 17 heads a kv head
    (512, 4, 1, 64, 513, 3, 16, BF, 1, "nhd"),       # 2048 rows, one kv head
    (3, 128, 16, 128, 4097, 100, 16, F16, 1, "nhd"), # few rows, spans across kv heads
    (24, 32, 8, 128, 6000, 300, 64, BF, 1, "hnd"),
]


@pytest.mark.parametrize("R,nq,nkv,hd,prefix,most,P,dt,chunk,layout", SHARED)
def test_shared_pass_matches_the_formula(C_, R, nq, nkv, hd, prefix, most, P, dt, chunk, layout):
    r = np.random.default_rng(R + prefix)
    lens = r.integers(0, most + 1, R)
    lens[0] = most
    if R > 3:
        lens[1], lens[2] = 0, 1
    s = make_attn(R + hd, R, nq, nkv, hd, prefix, lens, P, dt, chunk, layout)
    poison_tail(s)
    attn_close(attend(C_, s), s, hd ** -0.5)


@pytest.mark.parametrize("R,nq,hd", [(40, 16, 128), (20, 16, 128), (80, 16, 64)])
def test_shared_pass_with_rising_maxima_padding_and_in_place(C_, R, nq, hd):
    for dt in (BF, F16):
        s = make_attn(31, R, nq, 4, hd, 1500, np.arange(R) % 50, 16, dt)
        s["k"] *= (torch.arange(1, s["k"].shape[0] + 1, device="cuda").to(dt) / 16)[:, None, None, None]
        attn_close(attend(C_, s, scale=0.3), s, 0.3)
        s["q"][5] = float("nan")
        s["seq"][5] = -1
        out = attend(C_, s)
        live = [r for r in range(R) if r != 5]
        keep = {k: (v[live] if k in ("q", "lens", "seq") else v) for k, v in s.items()}
        attn_close(out[live], keep, hd ** -0.5)
        assert bool((out[5] == 5).all())
        again = attend(C_, s)
        assert torch.equal(again, out)
        s["q"][5] = 5.0
        attend(C_, s, out=s["q"])
        assert torch.equal(s["q"], out)


@pytest.mark.parametrize("R", [24, 90])
def test_shared_pass_bad_pages_nan_and_infinity(C_, R):
    s = make_attn(32, R, 16, 4, 128, 1333, np.full(R, 50), 16, BF)
    good = attend(C_, s)
    attn_close(good, s, 128 ** -0.5)
    s["tables"][1, 2] = s["k"].shape[0]
    s["lens"][3] = s["tables"].shape[1] * 16 + 1
    out = attend(C_, s)
    assert bool(torch.isnan(out[[1, 3]]).all())
    rest = [r for r in range(R) if r not in (1, 3)]
    assert torch.equal(out[rest], good[rest])
    keep = s["ptab"].clone()
    for bad in (-1, s["k"].shape[0], 1 << 30):
        for at in (0, 40, len(keep) - 1):
            s["ptab"].copy_(keep)
            s["ptab"][at] = bad
            assert bool(torch.isnan(attend(C_, s)).all())
    s["ptab"].copy_(keep)
    page = s["ptab"][50].long()
    s["v"][page, 3, 2] = float("inf")   # a value of kv head 2: its heads alone
    s["k"][s["ptab"][60].long(), 1, 0] = float("nan")
    out = attend(C_, s)
    assert bool(torch.isnan(out[rest][:, :4]).all()) and bool((~torch.isfinite(out[rest][:, 8:12])).all())
    assert torch.equal(out[rest][:, 4:8], good[rest][:, 4:8]) and torch.equal(out[rest][:, 12:], good[rest][:, 12:])


def test_shared_pass_queries_that_16_byte_loads_do_not_fit(C_):
    s = make_attn(33, 40, 16, 4, 128, 1200, np.full(40, 9), 16, F16)
    ref = attend(C_, s)
    wide = torch.zeros((40, 17, 130), device="cuda", dtype=F16)
    wide[:, 1:, 2:] = s["q"]
    assert torch.equal(attend(C_, {**s, "q": wide[:, 1:, 2:]}, out=torch.empty_like(s["q"])), ref)


def test_shared_pass_in_two_streams_at_once(C_):
    cases = [make_attn(40 + i, 64, 32, 8, (128, 64)[i % 2], 3000, np.full(64, 200), 32, (BF, F16)[i // 2]) for i in range(4)]
    want = [attend(C_, s) for s in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[torch.zeros_like(w) for _ in range(6)] for w in want]
    for i in range(6):
        for s, st, o in zip(cases, streams, got):
            with torch.cuda.stream(st):
                attend(C_, s, out=o[i])
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for os, w in zip(got, want) for o in os)


def test_attention_without_tables_of_its_own(C_):
    for R in (1, 3, 60):
        s = make_attn(50, R, 16, 4, 128, 900, np.zeros(R, np.int32), 16, BF)
        want = attend(C_, s)
        attn_close(want, s, 128 ** -0.5)
        none = {**s, "tables": torch.zeros((R, 0), device="cuda", dtype=torch.int32)}  # tables of no pages
        assert torch.equal(attend(C_, none), want)
        none["lens"] = torch.ones_like(s["lens"])  # a token that no table has
        assert bool(torch.isnan(attend(C_, none)).all())
        pad = {**s, "tables": torch.zeros((0, 4), device="cuda", dtype=torch.int32), "seq": torch.full_like(s["seq"], -1)}
        assert bool((attend(C_, pad) == 5).all())  # nothing but padding
        empty = {**s, "prefix": 0, "ptab": None}
        assert bool((attend(C_, empty) == 0).all())
