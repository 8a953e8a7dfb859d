"""The paged key-value cache operators, case by case: attention of new tokens over
the pages, attention over the pages a cheap score selects, eviction by accumulated
attention weight, and the rotary append with the pages' bounds.

`run` computes an operator from elementary torch operations, or, where `own` is
true, by the calls of expertrelay_b200.kv.
"""

from __future__ import annotations

import math

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
ES = {"f32": 4, "bf16": 2}
THETA = 1.0e6  # the rotary base of Qwen1.5-MoE


# ---- cases -------------------------------------------------------------------
def listed():
    return [
        # one sequence of Qwen1.5-MoE-A2.7B (16 heads of 128, fp32 cache) near the end of a 512-token prompt
        # and 128 new tokens: the smallest call, where latency counts
        {"name": "attend_one_f32", "op": "attend", "rows": 1, "kv_heads": 16, "group": 1, "dim": 128, "page": 16,
         "length": 639, "ragged": False, "cache": "f32", "query": "f32", "mass": False},
        # a serving batch of the same heads with a 16-bit cache, its sequences of odd and uneven lengths
        {"name": "attend_batch_bf16", "op": "attend", "rows": 48, "kv_heads": 16, "group": 1, "dim": 128, "page": 16,
         "length": 4097, "ragged": True, "cache": "bf16", "query": "bf16", "mass": False},
        # shared key heads, long contexts: the largest
        {"name": "attend_long_bf16", "op": "attend", "rows": 16, "kv_heads": 4, "group": 8, "dim": 128, "page": 64,
         "length": 65536, "ragged": False, "cache": "bf16", "query": "bf16", "mass": False},
        # one long sequence with few key heads: only the split over the length fills the card
        {"name": "attend_single_long", "op": "attend", "rows": 1, "kv_heads": 2, "group": 6, "dim": 64, "page": 32,
         "length": 131071, "ragged": False, "cache": "bf16", "query": "f32", "mass": False},
        # decode that also accumulates each position's attention weight, for the eviction below
        {"name": "attend_mass_bf16", "op": "attend", "rows": 8, "kv_heads": 8, "group": 4, "dim": 128, "page": 32,
         "length": 16000, "ragged": True, "cache": "bf16", "query": "bf16", "mass": True},
        # sparse decode of one long sequence: 64 of 2048 pages
        {"name": "sparse_one", "op": "sparse", "rows": 1, "kv_heads": 4, "group": 8, "dim": 128, "page": 32,
         "length": 65500, "ragged": False, "cache": "bf16", "query": "bf16", "budget": 64, "sinks": 1, "recent": 4},
        # sparse decode of a batch, uneven lengths, some of them inside the budget
        {"name": "sparse_batch", "op": "sparse", "rows": 32, "kv_heads": 8, "group": 4, "dim": 128, "page": 64,
         "length": 32768, "ragged": True, "cache": "bf16", "query": "bf16", "budget": 48, "sinks": 1, "recent": 2},
        # one sequence's fp32 cache cut to 1024 positions
        {"name": "evict_one_f32", "op": "evict", "rows": 1, "kv_heads": 16, "dim": 128, "page": 16, "length": 2501,
         "ragged": False, "cache": "f32", "budget": 1024, "sinks": 4, "recent": 128},
        # a batch of long sequences cut to 4096 positions each, two lengths under that among them
        {"name": "evict_batch_bf16", "op": "evict", "rows": 16, "kv_heads": 8, "dim": 128, "page": 64,
         "length": 32768, "ragged": True, "cache": "bf16", "budget": 4096, "sinks": 4, "recent": 512},
        # one decode step's rows of 64 sequences, at far positions
        {"name": "append_step_bf16", "op": "append", "rows": 64, "kv_heads": 16, "group": 1, "dim": 128, "page": 16,
         "length": 32000, "ragged": True, "new": 1, "cache": "bf16", "query": "bf16", "bounds": False},
        # prompts of 4 sequences, 16384 tokens in all, into a 16-bit cache with the pages' bounds
        {"name": "append_prompt_bf16", "op": "append", "rows": 4, "kv_heads": 16, "group": 1, "dim": 128, "page": 64,
         "length": 4096, "ragged": False, "new": 4096, "cache": "bf16", "query": "bf16", "bounds": True},
        # the same for an fp32 cache without bounds, shared key heads, an odd number of tokens
        {"name": "append_prompt_f32", "op": "append", "rows": 3, "kv_heads": 2, "group": 7, "dim": 64, "page": 24,
         "length": 1999, "ragged": False, "new": 1777, "cache": "f32", "query": "f32", "bounds": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    c = {"op": rng.choice(["attend", "attend", "sparse", "evict", "append"])}
    c["rows"] = _log(rng, 1, 64)
    c["kv_heads"] = rng.choice([1, 2, 3, 4, 8, 16])
    if c["op"] != "evict":
        c["group"] = rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 16])
    c["dim"] = rng.choice([32, 64, 80, 96, 128, 128, 128, 192, 256])
    c["page"] = rng.choice([8, 16, 16, 24, 32, 64, 64, 128])
    c["ragged"] = rng.random() < 0.6
    c["cache"] = rng.choice(["f32", "bf16", "bf16"])
    if c["op"] != "evict":
        c["query"] = "f32" if c["cache"] == "f32" else rng.choice(["f32", "bf16", "bf16"])
    # the cache stays under 2 GB (the plain forms hold it several times over in 32 bits)
    most = int(2e9 / (c["rows"] * c["kv_heads"] * c["dim"] * 2 * ES[c["cache"]]))
    c["length"] = _log(rng, 1, max(1, min(131072, most)))
    if c["op"] == "attend":
        c["mass"] = rng.random() < 0.3
    if c["op"] == "sparse":
        c["budget"] = _log(rng, 4, 128)
        c["sinks"], c["recent"] = rng.randint(0, 2), rng.randint(0, 2)
    if c["op"] == "evict":
        c["budget"] = _log(rng, 8, 8192)
        c["sinks"] = rng.randint(0, min(4, c["budget"] // 4))
        c["recent"] = rng.randint(0, c["budget"] // 2)
    if c["op"] == "append":
        c["length"] = min(c["length"], 32768)
        row = c["kv_heads"] * (c["group"] + 2) * c["dim"]  # values of one token's q|k|v
        c["new"] = 1 if rng.random() < 0.4 else _log(rng, 1, max(1, min(c["length"], int(1e8 / (row * c["rows"])))))
        c["bounds"] = rng.random() < 0.5
    return c


def _lengths(case):
    """Every sequence's length, from the case alone: all alike, or spread over 1 .. length with an idle (empty)
    sequence among five or more."""
    n, top = case["rows"], case["length"]
    if not case["ragged"]:
        return [top] * n
    got = [1 + int((i * 0.6180339887498949 + 0.37) % 1.0 * (top - 1) + 0.5) for i in range(n)]
    got[0] = top
    if n >= 5 and case["op"] != "append":
        got[3] = 0
    return got


def _width(case):
    return max(1, -(-case["length"] // case["page"]))


def work(case):
    es, kh, d = ES[case["cache"]], case["kv_heads"], case["dim"]
    lens, ps = _lengths(case), case["page"]
    row = kh * d * 2 * es  # one position's keys and values
    if case["op"] == "evict":
        kept = sum(min(n, case["budget"]) for n in lens)
        cut = sum(n for n in lens if n > case["budget"])
        return {"bytes": 2 * kept * row + 4 * kh * (cut + 2 * kept) + 4 * kh * kept + 4 * sum(-(-n // ps) for n in lens),
                "flops": 0}
    heads = kh * case["group"]
    if case["op"] == "append":
        new = sum(min(case["new"], n) for n in lens)
        moved = new * (heads + 2 * kh) * d * ES[case["query"]] + new * heads * d * ES[case["query"]] + new * row
        if case["bounds"]:  # the touched pages' old keys, their codes and scales
            first = [(n - min(case["new"], n)) // ps * ps for n in lens]
            moved += sum((n - min(case["new"], n) - f) * row // 2 for n, f in zip(lens, first))
            moved += sum((-(-n // ps) - f // ps) * kh * (2 * d + 4) for n, f in zip(lens, first))
        return {"bytes": moved, "flops": 3 * new * (heads + kh) * d}
    qo = 2 * case["rows"] * heads * d * ES[case["query"]]
    pages = [-(-n // ps) for n in lens]
    if case["op"] == "attend":
        total = sum(lens)
        return {"bytes": total * row + qo + 4 * sum(pages) + (8 * kh * total if case["mass"] else 0),
                "flops": 4 * d * heads * total}
    used = sum(min(n, case["budget"] * ps) for n in lens)
    # all pages' bounds, the last page's keys for its new bounds, and what the chosen pages hold
    last = sum((n - 1) % ps + 1 for n in lens if n) * row // 2
    chosen = kh * sum(min(p, case["budget"]) for p in pages)
    return {"bytes": sum(pages) * (kh * (2 * d + 4) + 4) + last + used * row + qo + 4 * chosen,
            "flops": 4 * d * heads * used + 2 * d * heads * sum(pages)}


# ---- inputs ------------------------------------------------------------------
def _pools(case, lens, gen, dev, spare=3):
    """Key and value pools with the sequences' pages strewn over them; slots that no sequence uses hold what an
    allocation may hold (NaN among it)."""
    ps, kh, d, dt = case["page"], case["kv_heads"], case["dim"], DT[case["cache"]]
    counts = [-(-n // ps) for n in lens]
    total = sum(counts) + spare
    k = torch.randn((total, kh, ps, d), generator=gen, device=dev, dtype=dt)
    v = torch.randn((total, kh, ps, d), generator=gen, device=dev, dtype=dt)
    # keys have a few strong channels, as trained ones do
    k *= (0.6 + 2.0 * torch.rand((1, kh, 1, d), generator=gen, device=dev) ** 6).to(dt)
    table = torch.full((len(lens), _width(case)), -1, dtype=torch.int32)
    order = torch.randperm(total, generator=gen, device=dev).cpu().to(torch.int32)
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = order[at:at + n]
        at += n
        if lens[s] % ps:
            k[int(table[s, n - 1]), :, lens[s] % ps:] = float("nan")
            v[int(table[s, n - 1]), :, lens[s] % ps:] = float("nan")
    return k, v, table.to(dev)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    lens = _lengths(case)
    st = {"case": dict(case), "lens": torch.tensor(lens, dtype=torch.int32, device=dev)}
    kh, d, ps = case["kv_heads"], case["dim"], case["page"]
    st["k"], st["v"], st["table"] = _pools(case, lens, gen, dev)
    if case["op"] in ("attend", "sparse"):
        st["q"] = torch.randn((case["rows"], kh * case["group"], d), generator=gen, device=dev).to(DT[case["query"]])
        st["scale"] = d ** -0.5
        if case["op"] == "attend" and case["mass"]:
            st["mass"] = torch.rand((case["rows"], kh, max(1, case["length"])), generator=gen, device=dev)
        if case["op"] == "sparse":
            shape = (st["k"].shape[0], kh, 2, d)
            st["codes"] = torch.zeros(shape, dtype=torch.int8, device=dev)
            st["scales"] = torch.zeros(shape[:2], device=dev)
            st["start"] = (st["lens"] - 1).clamp(min=0)  # this step's new position
            _bounds(st, st["lens"], torch.zeros_like(st["lens"]))
    elif case["op"] == "evict":
        # weight falls on few positions, and many later ones have received none yet (exact ties)
        w = torch.rand((case["rows"], kh, max(1, case["length"])), generator=gen, device=dev)
        st["mass"] = torch.where(w < 0.3, torch.zeros_like(w), w ** 8)
        width = -(-case["budget"] // ps)
        st["to_k"] = torch.zeros((case["rows"] * width, kh, ps, d), dtype=st["k"].dtype, device=dev)
        st["to_v"] = torch.zeros_like(st["to_k"])
        order = torch.randperm(case["rows"] * width, generator=gen, device=dev)
        st["to_table"] = order.to(torch.int32).reshape(case["rows"], width)
        st["to_mass"] = torch.zeros((case["rows"], kh, width * ps), device=dev)
    else:
        heads = kh * case["group"]
        rows, pos = [], []
        for s, n in enumerate(lens):
            new = min(case["new"], n)
            rows += [s] * new
            pos += range(n - new, n)
        st["seq"] = torch.tensor(rows, dtype=torch.int32, device=dev)
        st["pos"] = torch.tensor(pos, dtype=torch.int32, device=dev)
        st["qkv"] = torch.randn((len(rows), (heads + 2 * kh) * d), generator=gen, device=dev).to(DT[case["query"]])
        st["start"] = torch.tensor([n - min(case["new"], n) for n in lens], dtype=torch.int32, device=dev)
        if case["bounds"]:
            st["codes"] = torch.zeros((st["k"].shape[0], kh, 2, d), dtype=torch.int8, device=dev)
            st["scales"] = torch.zeros((st["k"].shape[0], kh), device=dev)
            at = [(s, p) for s, n in enumerate(lens) for p in range((n - min(case["new"], n)) // ps, -(-n // ps))]
            st["touched"] = st["table"].long()[tuple(torch.tensor(at, device=dev).T)]
    return st


# ---- one pass ----------------------------------------------------------------
def _handle(st):
    """The cache's handle, kept by a program as long as the cache."""
    if "handle" not in st:
        from expertrelay_b200 import kv

        st["handle"] = kv.PagedKV(st["k"], st["v"], st["table"])
        if "codes" in st:
            st["bounds"] = kv.PageBounds(st["codes"], st["scales"])
        if "to_k" in st:
            st["to"] = kv.PagedKV(st["to_k"], st["to_v"], st["to_table"])
    return st["handle"]


def run(st):
    case = st["case"]
    op = case["op"]
    if own:
        from expertrelay_b200 import kv

        cache = _handle(st)
        if op == "attend":
            out = kv.attend(cache, st["q"], st["lens"], mass=st.get("mass"))
            return {"out": out, "mass": st["mass"]} if case["mass"] else {"out": out}
        if op == "sparse":
            kv.page_bounds(cache, st["bounds"], st["lens"], st["start"])
            pages, counts = kv.select_pages(cache, st["bounds"], st["q"], st["lens"], case["budget"],
                                            sinks=case["sinks"], recent=case["recent"])
            out = kv.attend(cache, st["q"], st["lens"], pages=pages, counts=counts)
            return {"pages": pages, "counts": counts, "out": out}
        if op == "evict":
            kept, lens = kv.evict(cache, st["lens"], st["mass"], st["to"], st["to_mass"], case["budget"],
                                  sinks=case["sinks"], recent=case["recent"])
            return {"kept": kept, "lens": lens, "k": st["to_k"], "v": st["to_v"], "mass": st["to_mass"]}
        q = kv.append(cache, st["qkv"], st["pos"], case["kv_heads"] * case["group"], THETA, seqs=st["seq"])
        if case["bounds"]:
            kv.page_bounds(cache, st["bounds"], st["lens"], st["start"])
    else:
        if op == "attend":
            return _attend(st)
        if op == "sparse":
            _bounds(st, st["lens"], st["start"])
            return _sparse(st)
        if op == "evict":
            return _evict(st)
        q = _append(st)
        if case["bounds"]:
            _bounds(st, st["lens"], st["start"])
    out = {"q": q, "k": st["k"], "v": st["v"]}
    if case["bounds"]:  # the renewed bounds, as the values they stand for
        out["bounds"] = st["codes"][st["touched"]] * st["scales"][st["touched"]][..., None, None]
    return out


# ---- the plain forms ---------------------------------------------------------
def _rows_of(pool, table):
    """[pages, kv_heads, page, d] by a table [rows, w] -> [rows, kv_heads, w * page, d]"""
    rows, w = table.shape
    got = pool[table.long().clamp(min=0)].transpose(1, 2)
    return got.reshape(rows, pool.shape[1], w * pool.shape[2], pool.shape[3])


def _softmax_rows(q, k, v, scale, valid):
    """q [R, KH, G, d], k, v [R, KH, n, d], valid [R, KH, n] -> out [R, KH, G, d], weights [R, KH, G, n], 32 bits."""
    s = torch.matmul(q.float() * scale, k.float().transpose(2, 3))
    s = s.masked_fill(~valid[:, :, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == float("-inf"), torch.zeros_like(m), m))
    p = p.masked_fill(~valid[:, :, None], 0.0)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    return torch.matmul(p, v.float().masked_fill(~valid[..., None], 0.0)), p


def _attend(st):
    case = st["case"]
    kh, ps = case["kv_heads"], case["page"]
    k, v = _rows_of(st["k"], st["table"]), _rows_of(st["v"], st["table"])
    q = st["q"].reshape(case["rows"], kh, case["group"], case["dim"])
    at = torch.arange(st["table"].shape[1] * ps, device=q.device)
    valid = (at[None] < st["lens"][:, None])[:, None].expand(-1, kh, -1)
    out, p = _softmax_rows(q, k, v, st["scale"], valid)
    out = out.reshape(st["q"].shape).to(st["q"].dtype)
    if not case["mass"]:
        return {"out": out}
    st["mass"] += p.sum(2)[:, :, :st["mass"].shape[2]]
    return {"out": out, "mass": st["mass"]}


def _bounds(st, lens, start):
    """Renews the int8 bounds of the pages that hold the positions start .. lens - 1 of each sequence."""
    ps, table = st["k"].shape[2], st["table"]
    at = torch.arange(table.shape[1], device=table.device)
    touched = (at[None] >= (start // ps)[:, None]) & (at[None] * ps < lens[:, None]) & (start < lens)[:, None]
    seq, ordinal = touched.nonzero(as_tuple=True)
    page = table[seq, ordinal].long()
    keys = st["k"][page].float()  # [m, kv_heads, page, d]
    live = torch.arange(ps, device=table.device)[None] < (lens[seq] - ordinal * ps)[:, None]
    hi = keys.masked_fill(~live[:, None, :, None], float("-inf")).amax(2)
    lo = keys.masked_fill(~live[:, None, :, None], float("inf")).amin(2)
    scale = torch.maximum(hi.abs(), lo.abs()).amax(-1) / 127.0
    by = torch.where(scale == 0, torch.ones_like(scale), scale)[..., None]
    st["codes"][page] = torch.stack([torch.round(lo / by), torch.round(hi / by)], 2).to(torch.int8)
    st["scales"][page] = scale


def _sparse(st):
    case, lens, table = st["case"], st["lens"].long(), st["table"].long()
    kh, ps, budget = case["kv_heads"], case["page"], case["budget"]
    q = st["q"].reshape(case["rows"], kh, case["group"], case["dim"]).float()
    t = q.abs().amax(-1, keepdim=True) / 127.0
    c = torch.round(q / torch.where(t == 0, torch.ones_like(t), t))
    codes = st["codes"][table.clamp(min=0)].float().permute(0, 2, 3, 4, 1)  # [R, KH, 2, d, w]
    whole = torch.matmul(c.clamp(max=0), codes[:, :, 0]) + torch.matmul(c.clamp(min=0), codes[:, :, 1])  # whole numbers
    score = (whole * t).amax(2) * st["scales"][table.clamp(min=0)].transpose(1, 2)  # [R, KH, w]
    n = (lens + ps - 1) // ps
    at = torch.arange(table.shape[1], device=q.device)[None]
    forced = (at < case["sinks"]) | (at >= (n - case["recent"])[:, None])
    rank = score.double().masked_fill(score.isnan(), -1e300).masked_fill(forced[:, None], 1e300)
    rank = rank.masked_fill((at >= n[:, None])[:, None], float("-inf"))
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    counts = torch.minimum(n, torch.full_like(n, budget))
    slots = torch.arange(best.shape[-1], device=q.device)
    best = torch.where(slots < counts[:, None, None], best, table.shape[1]).sort(-1).values
    used = best < table.shape[1]
    pages = torch.full((case["rows"], kh, budget), -1, dtype=torch.int32, device=q.device)
    pages[..., :best.shape[-1]] = torch.where(used, best, -1).to(torch.int32)
    counts = counts[:, None].expand(-1, kh).to(torch.int32).contiguous()
    # attention over the pages chosen
    row = torch.arange(case["rows"], device=q.device)[:, None, None]
    head = torch.arange(kh, device=q.device)[None, :, None]
    page = table[row, best.clamp(max=table.shape[1] - 1)].clamp(min=0)
    shape = (case["rows"], kh, -1, case["dim"])
    pos = best[..., None] * ps + torch.arange(ps, device=q.device)
    valid = ((pos < lens[:, None, None, None]) & used[..., None]).reshape(case["rows"], kh, -1)
    out, _ = _softmax_rows(q, st["k"][page, head].reshape(shape), st["v"][page, head].reshape(shape), st["scale"], valid)
    return {"pages": pages, "counts": counts, "out": out.reshape(st["q"].shape).to(st["q"].dtype)}


def _evict(st):
    case, lens = st["case"], st["lens"].long()
    kh, ps, budget = case["kv_heads"], case["page"], case["budget"]
    n = st["mass"].shape[2]
    at = torch.arange(n, device=lens.device)[None]
    forced = (at < case["sinks"]) | (at >= (lens - case["recent"])[:, None])
    rank = st["mass"].double().masked_fill(st["mass"].isnan(), -1e300).masked_fill(forced[:, None], 1e300)
    rank = rank.masked_fill((at >= lens[:, None])[:, None], float("-inf"))
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    new = lens.clamp(max=budget)
    slots = torch.arange(best.shape[-1], device=lens.device)
    best = torch.where(slots < new[:, None, None], best, n).sort(-1).values
    kept = torch.full((case["rows"], kh, budget), -1, dtype=torch.int32, device=lens.device)
    kept[..., :best.shape[-1]] = torch.where(best < n, best, -1).to(torch.int32)
    seq, head, slot = (best < n).nonzero(as_tuple=True)
    src = best[seq, head, slot]
    page = st["table"].long()[seq, src // ps]
    to = st["to_table"].long()[seq, slot // ps]
    st["to_k"][to, head, slot % ps] = st["k"][page, head, src % ps]
    st["to_v"][to, head, slot % ps] = st["v"][page, head, src % ps]
    st["to_mass"][seq, head, slot] = st["mass"][seq, head, src]
    return {"kept": kept, "lens": new.to(torch.int32), "k": st["to_k"], "v": st["to_v"], "mass": st["to_mass"]}


def _append(st):
    case = st["case"]
    kh, d, ps = case["kv_heads"], case["dim"], case["page"]
    heads = kh * case["group"]
    x = st["qkv"].float().reshape(-1, heads + 2 * kh, d)
    j = torch.arange(d // 2, device=x.device, dtype=torch.float64)
    angle = st["pos"].double()[:, None] * THETA ** (-2.0 * j / d)  # 32 bits lose far positions
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    a, b = x[:, :heads + kh, :d // 2], x[:, :heads + kh, d // 2:]
    turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    pos = st["pos"].long()
    page = st["table"].long()[st["seq"].long(), pos // ps]
    st["k"][page, :, pos % ps] = turned[:, heads:].to(st["k"].dtype)
    st["v"][page, :, pos % ps] = x[:, heads + kh:].to(st["v"].dtype)
    return turned[:, :heads].to(st["qkv"].dtype)


# ---- the definitions in 64 bits ----------------------------------------------
def _exact_row(q, k, v, scale):
    """q [KH, G, d], k, v [KH, n, d] in 64 bits -> out [KH, G, d], weights [KH, G, n]"""
    if k.shape[1] == 0:
        return torch.zeros_like(q), q.new_zeros(q.shape[0], q.shape[1], 0)
    p = torch.softmax(torch.einsum("hgd,hnd->hgn", q, k) * scale, -1)
    return torch.einsum("hgn,hnd->hgd", p, v), p


def _exact_tokens(st, s, n):
    """Sequence s's first n keys and values, [KH, n, d] in 64 bits."""
    ps = st["k"].shape[2]
    pages = st["table"][s, : -(-n // ps)].long()
    return tuple(torch.cat(list(x[pages].double()), 1)[:, :n] if n else x.new_zeros(x.shape[1], 0, x.shape[3]).double()
                 for x in (st["k"], st["v"]))


def exact(case, seed):
    st = prepare(case, seed)
    lens, kh, ps, d = _lengths(case), case["kv_heads"], case["page"], case["dim"]
    table = st["table"].cpu().tolist()
    if case["op"] == "append":
        heads = kh * case["group"]
        x = st["qkv"].double().reshape(-1, heads + 2 * kh, d)
        k, v = st["k"].double(), st["v"].double()
        half = d // 2
        turn = torch.polar(torch.ones(x.shape[0], half, dtype=torch.float64, device=x.device),
                           st["pos"].double()[:, None] / THETA ** (torch.arange(half, device=x.device).double() * 2 / d))
        z = torch.view_as_real(torch.complex(x[..., :half], x[..., half:])[:, :heads + kh] * turn[:, None])
        z = torch.cat([z[..., 0], z[..., 1]], -1)
        at = 0
        for s, n in enumerate(lens):
            new = min(case["new"], n)
            pos = torch.arange(n - new, n, device=x.device)
            page = st["table"][s].long()[pos // ps]
            k[page, :, pos % ps] = z[at:at + new, heads:]
            v[page, :, pos % ps] = x[at:at + new, heads + kh:]
            at += new
        out = {"q": z[:, :heads], "k": k, "v": v}
        # the bounds go by the keys as they were rounded to the cache's type: no value in 64 bits
        return {**out, "bounds": None} if case["bounds"] else out
    if case["op"] == "evict":
        k, v, mass = st["to_k"].double(), st["to_v"].double(), st["to_mass"].double()
        kept = torch.full((case["rows"], kh, case["budget"]), -1, dtype=torch.int32)
        for s, n in enumerate(lens):
            m = min(n, case["budget"])
            if not m:
                continue
            ks, vs = _exact_tokens(st, s, n)
            for h in range(kh):
                order = list(range(n))
                if n > m:
                    first, last = case["sinks"], n - case["recent"]
                    w = st["mass"][s, h, first:last].double()
                    mid = (torch.sort(-w, stable=True).indices[: m - first - case["recent"]] + first).tolist()
                    order = sorted(list(range(first)) + mid + list(range(last, n)))
                pick = torch.tensor(order, device=k.device)
                slot = torch.arange(m, device=k.device)
                to = st["to_table"][s].long()[slot // ps]
                k[to, h, slot % ps], v[to, h, slot % ps] = ks[h, pick], vs[h, pick]
                mass[s, h, :m] = st["mass"][s, h, pick].double()
                kept[s, h, :m] = pick.to(torch.int32).cpu()
        return {"kept": kept, "lens": torch.tensor([min(n, case["budget"]) for n in lens], dtype=torch.int32), "k": k,
                "v": v, "mass": mass}
    q = st["q"].double().reshape(case["rows"], kh, case["group"], d)
    out = torch.zeros_like(q)
    if case["op"] == "attend":
        mass = st["mass"].double() if case["mass"] else None
        for r, n in enumerate(lens):
            out[r], p = _exact_row(q[r], *_exact_tokens(st, r, n), d ** -0.5)
            if mass is not None:
                mass[r, :, :n] += p.sum(1)
        out = out.reshape(st["q"].shape)
        return {"out": out, "mass": mass} if case["mass"] else {"out": out}
    pages = torch.full((case["rows"], kh, case["budget"]), -1, dtype=torch.int32)
    counts = torch.zeros((case["rows"], kh), dtype=torch.int32)
    for r, n in enumerate(lens):
        total = -(-n // ps)
        if not total:
            continue
        ks, vs = _exact_tokens(st, r, n)
        at = torch.tensor(table[r][:total], device=q.device)
        for h in range(kh):
            # the score as it is defined: whole numbers, then two products and a maximum in 32 bits
            qf = st["q"].reshape(q.shape)[r, h].float()
            t = qf.abs().amax(-1) / 127.0
            c = torch.round(qf / t[:, None]).nan_to_num(0.0).double()
            lo, hi = st["codes"][at, h, 0].double(), st["codes"][at, h, 1].double()
            whole = c.clamp(min=0) @ hi.T + c.clamp(max=0) @ lo.T
            score = (whole.float() * t[:, None]).amax(0) * st["scales"][at, h]
            order = list(range(total))
            if total > case["budget"]:
                first, last = case["sinks"], total - case["recent"]
                want = case["budget"] - first - case["recent"]
                mid = (torch.sort(-score[first:last], stable=True).indices[:want] + first).tolist()
                order = sorted(list(range(first)) + mid + list(range(last, total)))
            pos = torch.tensor([p * ps + i for p in order for i in range(ps) if p * ps + i < n], device=q.device)
            out[r, h] = _exact_row(q[r, h:h + 1], ks[h:h + 1, pos], vs[h:h + 1, pos], d ** -0.5)[0][0]
            pages[r, h, : len(order)] = torch.tensor(order, dtype=torch.int32)
            counts[r, h] = len(order)
    return {"pages": pages, "counts": counts, "out": out.reshape(st["q"].shape)}
