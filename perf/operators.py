"""Cases and plain forms of the paged-serving operators: page tables from request lengths, norms of
queries and keys with the position rotation, and attention of a batch that shares a long prefix.

``run`` computes an operator in elementary torch operations (``own`` false) or through the library's
entry points (``own`` true); ``exact`` computes it in 64 bits, written apart from the plain form.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # two requests a few tokens into their answers to a short system prompt: latency
        {"name": "attn_two_short", "op": "attn", "rows": 2, "q_heads": 28, "kv_heads": 4, "head_dim": 128,
         "prefix": 512, "own_max": 40, "page": 16, "dtype": "bf16", "chunk": 1},
        # a small batch on a 2k prompt
        {"name": "attn_batch8", "op": "attn", "rows": 8, "q_heads": 32, "kv_heads": 8, "head_dim": 128,
         "prefix": 2048, "own_max": 300, "page": 16, "dtype": "bf16", "chunk": 1},
        # odd sizes throughout: a prefix that ends inside a page and a tile, heads of 64 channels
        {"name": "attn_odd_hd64", "op": "attn", "rows": 37, "q_heads": 12, "kv_heads": 3, "head_dim": 64,
         "prefix": 5003, "own_max": 777, "page": 32, "dtype": "fp16", "chunk": 1},
        # several new tokens a request at once (a draft to verify), each row with its own length
        {"name": "attn_drafts", "op": "attn", "rows": 96, "q_heads": 32, "kv_heads": 8, "head_dim": 128,
         "prefix": 8192, "own_max": 1024, "page": 64, "dtype": "bf16", "chunk": 4},
        # the 32k context of the decode benchmark as the shared document of a large batch: the largest
        {"name": "attn_batch256_32k", "op": "attn", "rows": 256, "q_heads": 32, "kv_heads": 8, "head_dim": 128,
         "prefix": 32768, "own_max": 2048, "page": 32, "dtype": "bf16", "chunk": 1},
        # one decoded token whose float32 rows go to a cache engine's step: latency
        {"name": "rope_one_token", "op": "rope", "rows": 1, "q_heads": 32, "kv_heads": 8, "head_dim": 128,
         "rot": 128, "norm": True, "pages": False, "dtype": "bf16", "out": "fp32", "page": 16},
        # a decode batch written into its pages, some rows padding
        {"name": "rope_decode200", "op": "rope", "rows": 200, "q_heads": 28, "kv_heads": 4, "head_dim": 128,
         "rot": 128, "norm": True, "pages": True, "dtype": "fp16", "out": "fp16", "page": 16},
        # a prompt of a float32 model without norms, half of each head rotated
        {"name": "rope_prompt_fp32", "op": "rope", "rows": 4099, "q_heads": 12, "kv_heads": 3, "head_dim": 64,
         "rot": 32, "norm": False, "pages": False, "dtype": "fp32", "out": "fp32", "page": 16},
        # a 32k prompt into the pages: the largest
        {"name": "rope_prompt_32k", "op": "rope", "rows": 32768, "q_heads": 32, "kv_heads": 8, "head_dim": 128,
         "rot": 128, "norm": True, "pages": True, "dtype": "bf16", "out": "bf16", "page": 32},
        # a decode step of a small batch: one new token a request
        {"name": "tables_decode64", "op": "tables", "seqs": 64, "new_max": 1, "ctx_max": 2048, "page": 16,
         "ended": 0.05, "scarce": False},
        # a large batch of chunked prompts beside decoding requests, with too few free pages for all
        {"name": "tables_chunks1000", "op": "tables", "seqs": 1000, "new_max": 512, "ctx_max": 4096, "page": 32,
         "ended": 0.1, "scarce": True},
        # prompts of many requests at once: the largest
        {"name": "tables_prompts", "op": "tables", "seqs": 4096, "new_max": 1024, "ctx_max": 1024, "page": 16,
         "ended": 0.1, "scarce": False},
    ]


def _log(rng, lo, hi):
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "rope", "tables"])
    if op == "attn":
        hd = rng.choice([64, 128, 128])
        kv = rng.choice([1, 2, 3, 4, 8])
        c = {"op": "attn", "rows": _log(rng, 1, 300), "q_heads": kv * rng.choice([1, 2, 3, 4, 7, 8, 12]), "kv_heads": kv,
             "head_dim": hd, "prefix": _log(rng, 1, 33000), "own_max": _log(rng, 1, 3000),
             "page": rng.choice([16, 32, 64, 128]), "dtype": rng.choice(["bf16", "fp16"]),
             "chunk": rng.choice([1, 1, 1, 2, 5])}
        # no drawn case costs more than the largest listed one
        while c["rows"] * c["q_heads"] * hd * c["prefix"] > 256 * 32 * 128 * 32768 or c["rows"] * c["own_max"] * kv * hd > 256 * 2048 * 1024:
            c["rows"] = max(1, c["rows"] // 2)
        return c
    if op == "rope":
        hd = rng.choice([64, 128, 128, 256])
        kv = rng.choice([1, 2, 3, 4, 8])
        dt = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        c = {"op": "rope", "rows": _log(rng, 1, 32768), "q_heads": kv * rng.choice([1, 2, 4, 7]), "kv_heads": kv,
             "head_dim": hd, "rot": hd if rng.random() < 0.7 else hd // 2, "norm": rng.random() < 0.7,
             "pages": rng.random() < 0.6, "dtype": dt, "out": "fp32" if rng.random() < 0.25 else dt,
             "page": rng.choice([16, 32, 64])}
        if c["pages"]:
            c["out"] = dt
        while c["rows"] * (c["q_heads"] + 2 * kv) * hd * SIZE[dt] > 32768 * 48 * 128 * 2:
            c["rows"] = max(1, c["rows"] // 2)
        return c
    return {"op": "tables", "seqs": _log(rng, 1, 4096), "new_max": _log(rng, 1, 1024), "ctx_max": _log(rng, 1, 8192),
            "page": rng.choice([16, 32, 64, 128]), "ended": rng.choice([0.0, 0.05, 0.3]), "scarce": rng.random() < 0.3}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _lens(case, seed):
    """Own lengths of an attention case's rows, and the request of each: drawn on the host."""
    r = np.random.default_rng([seed, 1])
    rows, chunk, most = case["rows"], case["chunk"], case["own_max"]
    seqs = -(-rows // chunk)
    last = r.integers(1, most + 1, seqs)
    last[r.integers(0, seqs)] = most
    seq = np.arange(rows) // chunk
    back = np.minimum((seq + 1) * chunk, rows) - 1 - np.arange(rows)
    return np.maximum(last[seq] - back, 1).astype(np.int32), seq.astype(np.int32), last.astype(np.int32)


def _prepare_attn(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    lens, seq, last = _lens(case, seed)
    dt, P, hd, kv = DTYPES[case["dtype"]], case["page"], case["head_dim"], case["kv_heads"]
    npre, width = -(-case["prefix"] // P), -(-case["own_max"] // P)
    need = -(-last // P)
    pages = npre + int(need.sum()) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    at = np.concatenate([[0], np.cumsum(need)])
    pos = at[:-1, None] + np.arange(width)[None]
    pos = torch.from_numpy(np.where(np.arange(width)[None] < need[:, None], pos, -1)).to(DEV)
    tables = torch.where(pos >= 0, order[(pos.clamp(min=0) + npre)], torch.zeros_like(pos, dtype=torch.int32) - 1)
    # keys with a few strong channels, as projections have them, queries that reach logits of some units
    k = torch.randn((pages, P, kv, hd), generator=g, device=DEV, dtype=dt)
    k[..., :4] *= 3
    v = torch.randn((pages, P, kv, hd), generator=g, device=DEV, dtype=dt)
    q = torch.randn((case["rows"], case["q_heads"], hd), generator=g, device=DEV, dtype=dt)
    return {"op": "attn", "q": q, "k": k, "v": v, "prefix_table": order[:npre].contiguous(), "prefix": case["prefix"],
            "tables": tables.to(torch.int32).contiguous(), "lens": torch.from_numpy(lens).to(DEV),
            "seq": torch.from_numpy(seq).to(DEV) if case["chunk"] > 1 else None, "width": width,
            "out": torch.empty_like(q)}


def _prepare_rope(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt, T, hd, nq, kv = DTYPES[case["dtype"]], case["rows"], case["head_dim"], case["q_heads"], case["kv_heads"]
    qkv = torch.randn((T, (nq + 2 * kv) * hd), generator=g, device=DEV, dtype=dt)
    q, k, v = (x.view(T, -1, hd) for x in qkv.split([nq * hd, kv * hd, kv * hd], dim=1))
    s = {"op": "rope", "q": q, "k": k, "v": v, "norm": case["norm"], "pages": case["pages"], "rot": case["rot"], "eps": 1e-6}
    s["qw"], s["kw"] = ((1 + 0.2 * torch.randn(hd, generator=g, device=DEV)).to(dt) for _ in range(2))
    most = 4 * T + 64
    inv = 1e6 ** (-torch.arange(0, case["rot"], 2, device=DEV, dtype=torch.float64) / case["rot"])
    ang = torch.arange(most, device=DEV, dtype=torch.float64)[:, None] * inv[None]
    s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    start = int(torch.randint(0, 3 * T + 64, (1,), generator=g, device=DEV))
    s["positions"] = torch.arange(start, start + T, device=DEV, dtype=torch.int32)
    odt = DTYPES[case["out"]]
    s["q_out"] = torch.zeros((T, nq, hd), device=DEV, dtype=odt)
    if case["pages"]:
        P = case["page"]
        n = -(-T // P) + 2
        slots = torch.randperm(n, generator=g, device=DEV)[:, None] * P + torch.arange(P, device=DEV)[None]
        slots = slots.reshape(-1)[:T].clone()
        slots[torch.rand(T, generator=g, device=DEV) < 0.02] = -1  # rows of padding
        s["slots"] = slots
        s["k_dst"], s["v_dst"] = (torch.zeros((n, P, kv, hd), device=DEV, dtype=dt) for _ in range(2))
    else:
        s["slots"] = None
        s["k_dst"], s["v_dst"] = (torch.zeros((T, kv, hd), device=DEV, dtype=odt) for _ in range(2))
    return s


def _new_lens(case):
    """New tokens of a tables case's requests before some end or rest: few long chunks, many short ones."""
    B = case["seqs"]
    return np.maximum(1, (((np.arange(B) + 0.5) / B) ** 2 * case["new_max"]).astype(np.int64))


def _tables_host(case, seed):
    r = np.random.default_rng([seed, 2])
    B, P = case["seqs"], case["page"]
    ctx = r.integers(0, case["ctx_max"] + 1, B)
    new = r.permutation(_new_lens(case))
    new[r.random(B) < case["ended"]] = -1
    new[r.random(B) < 0.02] = 0
    held = -(-ctx // P)
    need = np.where(new > 0, -(-(ctx + np.maximum(new, 0)) // P) - held, 0)
    return ctx.astype(np.int32), new.astype(np.int32), held, need


def _prepare_tables(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    ctx, new, held, need = _tables_host(case, seed)
    B, P = case["seqs"], case["page"]
    width = -(-(case["ctx_max"] + case["new_max"]) // P)
    free = int(need.sum() * (0.6 if case["scarce"] else 1.1)) + 1
    total = B * width + B * width // 5 + 16  # the pool; what is neither held nor free belongs to others
    order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    at = torch.from_numpy(np.concatenate([[0], np.cumsum(held)])[:-1]).to(DEV)
    j = torch.arange(width, device=DEV)[None]
    has = j < torch.from_numpy(held).to(DEV)[:, None]
    tables = torch.where(has, order[torch.where(has, at[:, None] + j, 0)], torch.full((), -1, device=DEV, dtype=torch.int32))
    fp = torch.full((total,), -1, device=DEV, dtype=torch.int32)
    fp[:free] = order[total - free:]
    rows = max(64, -(-int(_new_lens(case).sum()) // 64) * 64)  # the row buffers are as large as any step of this batch
    e = lambda n, dt=torch.int32: torch.zeros(n, device=DEV, dtype=dt)  # noqa: E731
    return {"op": "tables", "ctx": torch.from_numpy(ctx).to(DEV), "new": torch.from_numpy(new).to(DEV), "tables": tables.contiguous(),
            "free_pages": fp, "free_count": torch.full((1,), free, device=DEV, dtype=torch.int32), "page": P, "offset": 100,
            "free_count_out": e(1), "seq_lens": e(B), "cu_new": e(B + 1), "slots": e(rows, torch.int64),
            "positions": e(rows), "row_seq": e(rows), "row_lens": e(rows), "deferred": e(1)}


def prepare(case, seed):
    return {"attn": _prepare_attn, "rope": _prepare_rope, "tables": _prepare_tables}[case["op"]](case, seed)


# ---------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------
def _plain_attn(s):
    q, P, width = s["q"].float(), s["k"].shape[1], s["width"]
    R, nq, hd = q.shape
    kv = s["k"].shape[2]
    kf, vf = s["k"].view(-1, kv, hd), s["v"].view(-1, kv, hd)
    t = torch.arange(s["prefix"], device=DEV)
    slot = s["prefix_table"].long()[t // P] * P + t % P
    kp, vp = kf[slot].float(), vf[slot].float()                        # [Lp, kv, hd]
    qg = q.view(R, kv, nq // kv, hd)
    sp = torch.matmul(qg.permute(1, 0, 2, 3).reshape(kv, -1, hd), kp.permute(1, 2, 0))
    sp = sp.view(kv, R, nq // kv, -1).transpose(0, 1)                  # [R, kv, g, Lp]
    t = torch.arange(width * P, device=DEV)
    tab = s["tables"].long() if s["seq"] is None else s["tables"].long()[s["seq"].long()]
    slot = tab[:, t // P] * P + t % P                                   # [R, W*P]
    live = t[None] < s["lens"][:, None]
    slot = torch.where(live, slot, 0)
    ko, vo = kf[slot].float(), vf[slot].float()                        # [R, W*P, kv, hd]
    so = torch.matmul(qg, ko.permute(0, 2, 3, 1))                      # [R, kv, g, W*P]
    so = so.masked_fill(~live[:, None, None], float("-inf"))
    w = torch.cat([sp, so], dim=-1) * (1.0 / math.sqrt(hd))
    w = torch.exp(w - w.amax(dim=-1, keepdim=True))
    w = w / w.sum(dim=-1, keepdim=True)
    wp, wo = w.split([sp.shape[-1], so.shape[-1]], dim=-1)
    o = torch.matmul(wp.transpose(0, 1).reshape(kv, -1, wp.shape[-1]), vp.transpose(0, 1))
    o = o.view(kv, R, nq // kv, hd).transpose(0, 1) + torch.matmul(wo, vo.transpose(1, 2))
    s["out"].copy_(o.reshape(R, nq, hd))
    return s["out"]


def _turn(x, w, s, c, sn):
    x = x.float()
    if s["norm"]:
        x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + s["eps"]) * w.float()
    h = s["rot"] // 2
    a, b, rest = x[..., :h], x[..., h:2 * h], x[..., 2 * h:]
    return torch.cat([a * c - b * sn, b * c + a * sn, rest], dim=-1)


def _plain_rope(s):
    p = s["positions"].long()
    c, sn = s["cos"][p][:, None], s["sin"][p][:, None]
    q, k = _turn(s["q"], s["qw"], s, c, sn), _turn(s["k"], s["kw"], s, c, sn)
    kd, vd = s["k_dst"], s["v_dst"]
    if s["slots"] is None:
        s["q_out"].copy_(q)
        kd.copy_(k)
        vd.copy_(s["v"])
    else:
        live = s["slots"] >= 0
        at = s["slots"][live]
        s["q_out"][live] = q[live].to(s["q_out"].dtype)
        kd.view(-1, *kd.shape[2:])[at] = k[live].to(kd.dtype)
        vd.view(-1, *vd.shape[2:])[at] = s["v"][live]
    return [s["q_out"], kd, vd]


def _plain_tables(s):
    P, tables = s["page"], s["tables"]
    B, W = tables.shape
    cap, rows = s["free_pages"].shape[0], s["slots"].shape[0]
    ctx, new = s["ctx"].long().clamp(min=0), s["new"].long().clamp(min=-1)
    ended, n = new < 0, new.clamp(min=0)
    held = (ctx + P - 1) // P
    # ended requests' pages go back on the stack, in request order
    back = torch.where(ended, held.clamp(max=W), 0)
    free0 = s["free_count"].long().clamp(0, cap)
    j = torch.arange(W, device=DEV)[None]
    to = free0 + (torch.cumsum(back, 0) - back)[:, None] + j
    to = torch.where((j < back[:, None]) & (to < cap), to, cap)
    grown = torch.cat([s["free_pages"], s["free_pages"][:1]])
    grown.scatter_(0, to.reshape(-1), tables.reshape(-1))
    s["free_pages"].copy_(grown[:cap])
    top = (free0 + back.sum()).clamp(max=cap)
    # rows, and what does not fit
    cu = torch.cumsum(n, 0)
    s["cu_new"][0] = 0
    s["cu_new"][1:] = cu
    last = (ctx + n + P - 1) // P
    wide = (n > 0) & ((last > W) | (cu > rows))
    need = torch.where((n > 0) & ~wide, last - held, 0)
    got = torch.cumsum(need, 0)
    late = wide | ((need > 0) & (got > top))
    given = torch.where(late, 0, need)
    s["free_count_out"].copy_((top - given.sum()).reshape(1))
    first = got - need
    at = (top - 1 - first[:, None] - (j - held[:, None])).clamp(0, cap - 1)
    fresh = (j >= held[:, None]) & (j < (held + given)[:, None])
    tables.copy_(torch.where(fresh, s["free_pages"][at], tables))
    s["seq_lens"].copy_(torch.where(ended, 0, torch.where(late, ctx, ctx + n)))
    s["deferred"].copy_(late.sum().reshape(1))
    # one entry a row
    t = torch.arange(rows, device=DEV)
    b = torch.searchsorted(cu, t, right=True)
    live = b < B
    b = b.clamp(max=B - 1)
    live = live & ~late[b]
    pos = torch.where(live, ctx[b] + t - (cu - n)[b], 0)
    slot = tables[b, pos // P].long() * P + pos % P
    s["slots"].copy_(torch.where(live, slot, -1))
    s["positions"].copy_(torch.where(live, pos + s["offset"], 0))
    s["row_seq"].copy_(torch.where(live, b, -1))
    s["row_lens"].copy_(torch.where(live, pos + 1, 0))
    return _tables_out(s)


def _tables_out(s):
    return [s[k] for k in ("tables", "free_pages", "free_count_out", "seq_lens", "cu_new", "slots", "positions", "row_seq",
                           "row_lens", "deferred")]


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    s = state
    if own:
        from tritiercache_b200 import _C
        if s["op"] == "attn":
            _C.shared_prefix_attention(s["q"], s["k"], s["v"], s["prefix_table"], s["prefix"], s["tables"], s["lens"], s["out"],
                                       row_seq=s["seq"])
            return s["out"]
        if s["op"] == "rope":
            w = (s["qw"], s["kw"]) if s["norm"] else (None, None)
            _C.qk_norm_rope(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["q_out"], s["k_dst"], s["v_dst"], q_weight=w[0],
                            k_weight=w[1], eps=s["eps"], positions=s["positions"], slots=s["slots"])
            return [s["q_out"], s["k_dst"], s["v_dst"]]
        _C.page_tables(s["ctx"], s["new"], s["tables"], s["free_pages"], s["free_count"], s["page"], s["seq_lens"], s["cu_new"],
                       s["slots"], s["positions"], s["row_seq"], s["row_lens"], s["deferred"],
                       free_count_out=s["free_count_out"], position_offset=s["offset"])
        return _tables_out(s)
    return {"attn": _plain_attn, "rope": _plain_rope, "tables": _plain_tables}[s["op"]](s)


def work(case):
    if case["op"] == "attn":
        lens, _, last = _lens(case, 0)
        kv, hd, nq, e = case["kv_heads"], case["head_dim"], case["q_heads"], SIZE[case["dtype"]]
        tokens = case["prefix"] + int(last.sum())
        return {"bytes": 2 * tokens * kv * hd * e + 2 * case["rows"] * nq * hd * e,
                "flops": 4 * nq * hd * (case["rows"] * case["prefix"] + int(lens.sum()))}
    if case["op"] == "rope":
        n = case["rows"] * (case["q_heads"] + 2 * case["kv_heads"]) * case["head_dim"]
        live = 0.98 if case["pages"] else 1.0
        return {"bytes": live * (n * (SIZE[case["dtype"]] + SIZE[case["out"]]) + case["rows"] * case["rot"] * 4),
                "flops": 8 * n}
    ctx, new, held, need = _tables_host(case, 0)
    rows = int(np.maximum(new, 0).sum())
    return {"bytes": 16 * case["seqs"] + 8 * int(need.sum()) + 8 * int(held[new < 0].sum()) + 20 * rows, "flops": 4 * rows}


# ---------------------------------------------------------------------------------------------
# in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "rope":
        res = []
        ang = [s["cos"][s["positions"].long()].double(), s["sin"][s["positions"].long()].double()]
        z = torch.complex(ang[0], ang[1])[:, None]
        h = s["rot"] // 2
        for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
            x = x.double()
            if s["norm"]:
                x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + s["eps"]) * w.double()
            y = torch.complex(x[..., :h], x[..., h:2 * h]) * z
            x = x.clone()
            x[..., :h], x[..., h:2 * h] = y.real, y.imag
            res.append(x)
        res.append(s["v"].double())
        if s["slots"] is None:
            return res
        live = torch.nonzero(s["slots"] >= 0).flatten()
        got = [torch.zeros(s["q_out"].shape, device=DEV, dtype=torch.float64).index_copy_(0, live, res[0][live])]
        for x in res[1:]:
            d = torch.zeros(s["k_dst"].shape, device=DEV, dtype=torch.float64)
            d.view(-1, *d.shape[2:]).index_copy_(0, s["slots"][live], x[live])
            got.append(d)
        return got
    P, kv, hd = s["k"].shape[1:]
    g = case["q_heads"] // kv
    out = torch.empty(s["q"].shape, device=DEV, dtype=torch.float64)
    pre = s["prefix_table"].long()
    kp, vp = (x[pre].reshape(-1, kv, hd)[:case["prefix"]].double() for x in (s["k"], s["v"]))
    lens, seq, _ = _lens(case, seed)
    for r in range(case["rows"]):
        own_pages = s["tables"][int(seq[r])][: -(-int(lens[r]) // P)].long()
        ks, vs = (x[own_pages].reshape(-1, kv, hd)[:int(lens[r])].double() for x in (s["k"], s["v"]))
        q = s["q"][r].double().view(kv, g, hd) / math.sqrt(hd)
        a = torch.cat([torch.einsum("hgd,thd->hgt", q, kp), torch.einsum("hgd,thd->hgt", q, ks)], dim=2)
        w = torch.softmax(a, dim=2)
        o = torch.einsum("hgt,thd->hgd", w[..., :case["prefix"]], vp) + torch.einsum("hgt,thd->hgd", w[..., case["prefix"]:], vs)
        out[r] = o.reshape(-1, hd)
    return out
