"""Operators of decoding with several continuations at once, case by case: attention for
a tree of drafted tokens over the paged cache, copying pages of all layers (forks) and
moving kept places together (accepted drafts), and beam search's selection.

`run` computes an operator from elementary torch operations, or, where `own` is
true, by the calls of expertrelay_b200.kv and expertrelay_b200.beam.
"""

from __future__ import annotations

import math

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
ES = {"f32": 4, "bf16": 2}
VOCAB = 151936  # of Qwen1.5-MoE


# ---- cases -------------------------------------------------------------------
def listed():
    return [
        # one sequence of Qwen1.5-MoE-A2.7B (16 heads of 128, fp32 cache) and a draft of 8 tokens, near the end of a
        # 512-token prompt and 128 new tokens: the smallest call, where latency counts
        {"name": "tree_one_f32", "op": "tree", "trees": 1, "nodes": 8, "shape": "tree", "kv_heads": 16, "group": 1,
         "dim": 128, "page": 16, "length": 631, "ragged": False, "cache": "f32", "query": "f32"},
        # a serving batch of the same heads with a 16-bit cache: uneven contexts (an empty one), uneven drafts
        {"name": "tree_batch_bf16", "op": "tree", "trees": 24, "nodes": 23, "shape": "tree", "kv_heads": 16, "group": 1,
         "dim": 128, "page": 16, "length": 4097, "ragged": True, "cache": "bf16", "query": "bf16"},
        # shared key heads, wide drafts, long contexts: the largest
        {"name": "tree_long_bf16", "op": "tree", "trees": 8, "nodes": 64, "shape": "tree", "kv_heads": 4, "group": 8,
         "dim": 128, "page": 64, "length": 32768, "ragged": False, "cache": "bf16", "query": "bf16"},
        # one long sequence with few key heads and a drafted chain: only the split over the length fills the card
        {"name": "tree_single_long", "op": "tree", "trees": 1, "nodes": 16, "shape": "chain", "kv_heads": 2, "group": 6,
         "dim": 64, "page": 32, "length": 131071, "ragged": False, "cache": "bf16", "query": "f32"},
        # a few sequences with fp32 caches and drafts of up to 37 tokens
        {"name": "tree_batch_f32", "op": "tree", "trees": 6, "nodes": 37, "shape": "tree", "kv_heads": 16, "group": 1,
         "dim": 128, "page": 24, "length": 2500, "ragged": True, "cache": "f32", "query": "f32"},
        # a beam step's forks: the last, partly filled pages of 4 beams, all 24 layers
        {"name": "copy_fork_f32", "op": "copy", "layers": 24, "pages": 4, "partial": True, "kv_heads": 16, "dim": 128,
         "page": 64, "cache": "f32"},
        # whole sequences copied, or a pool's pages moved to its front
        {"name": "copy_many_bf16", "op": "copy", "layers": 8, "pages": 500, "partial": False, "kv_heads": 8, "dim": 128,
         "page": 64, "cache": "bf16"},
        # one sequence's accepted path of up to 5 of 8 drafted tokens, all 24 layers
        {"name": "accept_one_f32", "op": "compact", "layers": 24, "rows": 1, "span": 8, "keep": 5, "accept": True,
         "kv_heads": 16, "dim": 128, "page": 16, "length": 631, "cache": "f32"},
        # a scattered part cut out of a batch's texts: the rest moves up
        {"name": "compact_batch_bf16", "op": "compact", "layers": 12, "rows": 12, "span": 1999, "keep": 1501,
         "accept": False, "kv_heads": 4, "dim": 128, "page": 32, "length": 77, "cache": "bf16"},
        # 4 beams of one text, two candidates a beam: latency counts
        {"name": "beam_one_f32", "op": "beam", "batch": 1, "beams": 4, "vocab": VOCAB, "count": 8, "logits": "f32",
         "first": False},
        # a batch of beam searches over 16-bit logits
        {"name": "beam_batch_bf16", "op": "beam", "batch": 32, "beams": 8, "vocab": VOCAB, "count": 16,
         "logits": "bf16", "first": False},
        # an odd vocabulary (rows that start anywhere), many beams, the search's first step (one live beam)
        {"name": "beam_odd_f32", "op": "beam", "batch": 7, "beams": 20, "vocab": 50257, "count": 40, "logits": "f32",
         "first": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    c = {"op": rng.choice(["tree", "tree", "tree", "copy", "compact", "beam"])}
    if c["op"] == "beam":
        c["vocab"] = _log(rng, 100, 200000)
        c["beams"] = _log(rng, 1, 32)
        c["batch"] = _log(rng, 1, max(1, min(64, int(4e7 / (c["vocab"] * c["beams"])))))
        c["count"] = min(c["beams"] * rng.choice([1, 2, 2, 3]), 64, c["vocab"])
        c["logits"] = rng.choice(["f32", "f32", "bf16"])
        c["first"] = rng.random() < 0.2
        return c
    c["kv_heads"] = rng.choice([1, 2, 3, 4, 8, 16])
    c["dim"] = rng.choice([32, 64, 80, 96, 128, 128, 128, 192, 256])
    c["page"] = rng.choice([8, 16, 16, 24, 32, 64, 64, 128])
    c["cache"] = rng.choice(["f32", "bf16", "bf16"])
    row = 2 * c["kv_heads"] * c["dim"] * ES[c["cache"]]  # a place's key and value in one layer
    if c["op"] == "tree":
        c["group"] = rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 16])
        c["query"] = "f32" if c["cache"] == "f32" else rng.choice(["f32", "bf16", "bf16"])
        c["trees"] = _log(rng, 1, 32)
        c["nodes"] = _log(rng, 1, 128 if c["group"] <= 8 else 64)
        c["shape"] = rng.choice(["tree", "tree", "chain"])
        c["ragged"] = rng.random() < 0.6
        # the contexts stay under 0.5 GB and, with their queries, under the largest listed case's products (one
        # tree's scores under 1.6 GB, which the plain form holds)
        most = min(5e8 / (c["trees"] * row), 4e8 / (c["nodes"] * c["kv_heads"] * c["group"]),
                   2.6e11 / (4 * c["trees"] * c["nodes"] * c["kv_heads"] * c["group"] * c["dim"]))
        c["length"] = _log(rng, 1, max(1, min(131072, int(most))))
        return c
    c["layers"] = rng.choice([1, 2, 6, 12, 24])
    if c["op"] == "copy":
        c["partial"] = rng.random() < 0.5
        c["pages"] = _log(rng, 1, max(1, min(512, int(5e8 / (c["layers"] * c["page"] * row)))))
        return c
    c["accept"] = rng.random() < 0.6
    c["rows"] = _log(rng, 1, 32)
    most = max(8, min(128 if c["accept"] else 4096, int(6e8 / (c["layers"] * c["rows"] * row))))
    c["span"] = _log(rng, 4, most)
    c["keep"] = _log(rng, 1, max(1, c["span"] // 4 if c["accept"] else c["span"] - 2))
    c["length"] = _log(rng, 1, 512)
    return c


def _spread(n, top, low):
    """n numbers over low .. top from nothing but n: the first is the top, the fourth of five or more the lowest."""
    got = [low + int((i * 0.6180339887498949 + 0.37) % 1.0 * (top - low) + 0.5) for i in range(n)]
    got[0] = top
    if n >= 5:
        got[3] = low
    return got


def _contexts(case):
    return _spread(case["trees"], case["length"], 0) if case["ragged"] else [case["length"]] * case["trees"]


def _nodes(case):
    return _spread(case["trees"], case["nodes"], 1)[::-1] if case["ragged"] else [case["nodes"]] * case["trees"]


def _parents(case, tree, n):
    """Parents within a tree of n nodes (-1: the text's last token): a chain, or a tree that branches anywhere,
    from its root too."""
    if case["shape"] == "chain":
        return list(range(-1, n - 1))
    return [max(-1, min(i - 1, int(((i + 3 * tree) * 0.7548776662466927) % 1.0 * (i + 0.2) + 0.3) - 1)) if i else -1
            for i in range(n)]


def _counts(case):
    """How many places each sequence keeps; of a batch of accepted drafts, none for one."""
    got = _spread(case["rows"], case["keep"], 1)
    if case["accept"] and case["rows"] >= 5:
        got[3] = 0
    return got


def _used(case):
    """Slots of each page that hold something."""
    return _spread(case["pages"], case["page"], 1)[::-1] if case["partial"] else [case["page"]] * case["pages"]


def work(case):
    op = case["op"]
    if op == "beam":
        b, k = case["batch"], case["count"]
        n = b * case["beams"] * case["vocab"]
        return {"bytes": n * ES[case["logits"]] + 4 * b * case["beams"] + 12 * b * k, "flops": 4 * n}
    row = 2 * case["kv_heads"] * case["dim"] * ES[case["cache"]]
    if op == "copy":
        return {"bytes": 2 * sum(_used(case)) * case["layers"] * row + 12 * case["pages"], "flops": 0}
    if op == "compact":
        counts = _counts(case)
        moved = sum(max(0, n - 1) if case["accept"] else n for n in counts)
        return {"bytes": 2 * moved * case["layers"] * row + 4 * sum(counts) + 16 * case["rows"], "flops": 0}
    heads = case["kv_heads"] * case["group"]
    ctx, nodes = _contexts(case), _nodes(case)
    seen = 0  # (node, key) pairs
    for t, (n, m) in enumerate(zip(ctx, nodes)):
        depth = []
        for p in _parents(case, t, m):
            depth.append(1 + (depth[p] if p >= 0 else 0))
        seen += m * n + sum(depth)
    pages = sum(-(-(n + m) // case["page"]) for n, m in zip(ctx, nodes))
    io = sum(nodes) * (2 * heads * case["dim"] * ES[case["query"]] + 4)
    return {"bytes": sum(n + m for n, m in zip(ctx, nodes)) * row + io + 4 * pages + 8 * case["trees"],
            "flops": 4 * case["dim"] * heads * seen}


# ---- inputs ------------------------------------------------------------------
def _tables(lens, ps, gen, spare=3):
    """A page table with the sequences' pages strewn over a pool, and the pool's size."""
    counts = [-(-n // ps) for n in lens]
    total = sum(counts) + spare
    table = torch.full((len(lens), max(1, *counts)), -1, dtype=torch.int32)
    order = torch.randperm(total, generator=gen, device=gen.device).cpu().to(torch.int32)
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = order[at:at + n]
        at += n
    return table, total


def _pool(shape, dtype, gen):
    """Keys and values; keys have a few strong channels, as trained ones do."""
    k = torch.randn(shape, generator=gen, device=gen.device, dtype=dtype)
    v = torch.randn(shape, generator=gen, device=gen.device, dtype=dtype)
    k *= (0.6 + 2.0 * torch.rand((shape[-3], 1, shape[-1]), generator=gen, device=gen.device) ** 6).to(dtype)
    return k, v


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    st = {"case": dict(case)}
    if case["op"] == "beam":
        b, m, n = case["batch"], case["beams"], case["vocab"]
        x = torch.randn((b * m, n), generator=gen, device=dev) * 2.5
        x[:, torch.randperm(n, generator=gen, device=dev)[: n // 500]] = float("-inf")  # tokens never to be chosen
        st["logits"] = x.to(DT[case["logits"]])
        st["scores"] = -12.0 * torch.rand((b, m), generator=gen, device=dev)
        if case["first"]:
            st["scores"][:, 1:] = float("-inf")
            st["scores"][:, 0] = 0.0
        return st
    dt, kh, ps, d = DT[case["cache"]], case["kv_heads"], case["page"], case["dim"]
    if case["op"] == "copy":
        n = case["pages"]
        total = 2 * n + 2
        st["k"], st["v"] = _pool((case["layers"], total, kh, ps, d), dt, gen)
        order = torch.randperm(total, generator=gen, device=dev).to(torch.int32)
        st["src"], st["dst"] = order[:n].clone(), order[n:2 * n].clone()
        st["used"] = torch.tensor(_used(case), dtype=torch.int32, device=dev) if case["partial"] else None
        return st
    if case["op"] == "compact":
        rows, span = case["rows"], case["span"]
        lens = [1 + (case["length"] * (i + 1)) // rows for i in range(rows)]
        table, total = _tables([n + span for n in lens], ps, gen)
        st["k"], st["v"] = _pool((case["layers"], total, kh, ps, d), dt, gen)
        st["table"] = table.to(dev)
        st["start"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        keep = torch.full((rows, case["keep"]), -1, dtype=torch.int32)
        counts = _counts(case)
        for i, n in enumerate(counts):
            # a path from the draft's first token on, or whatever lies behind the first cut
            lead = 1 if case["accept"] else min(2, span - n)
            at = torch.randperm(span - lead, generator=gen, device=dev)[: n - 1 if case["accept"] and n else n].cpu()
            at = torch.sort(at + lead).values
            keep[i, :n] = torch.cat([torch.zeros(1, dtype=at.dtype), at])[:n] if case["accept"] else at
        st["keep"], st["counts"] = keep.to(dev), torch.tensor(counts, dtype=torch.int32, device=dev)
        return st
    ctx, nodes = _contexts(case), _nodes(case)
    lens = [n + m for n, m in zip(ctx, nodes)]
    table, total = _tables(lens, ps, gen)
    st["k"], st["v"] = _pool((total, kh, ps, d), dt, gen)
    for s, n in enumerate(lens):  # slots that no sequence uses hold what an allocation may hold
        if n % ps:
            st["k"][int(table[s, n // ps]), :, n % ps:] = float("nan")
            st["v"][int(table[s, n // ps]), :, n % ps:] = float("nan")
    st["table"], st["lens"] = table.to(dev), torch.tensor(ctx, dtype=torch.int32, device=dev)
    starts = [0]
    for m in nodes:
        starts.append(starts[-1] + m)
    st["starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    parents = [p for t, m in enumerate(nodes) for p in _parents(case, t, m)]
    st["parents"] = torch.tensor(parents, dtype=torch.int32, device=dev)
    st["q"] = torch.randn((starts[-1], kh * case["group"], d), generator=gen, device=dev).to(DT[case["query"]])
    st["scale"] = d ** -0.5
    return st


# ---- one pass ----------------------------------------------------------------
def _handle(st):
    """The cache's handle, kept by a program as long as the cache."""
    if "handle" not in st:
        from expertrelay_b200 import kv

        if st["case"]["op"] == "tree":
            st["handle"] = kv.PagedKV(st["k"], st["v"], st["table"])
        else:
            table = st["table"] if "table" in st else torch.zeros((1, 1), dtype=torch.int32, device=st["k"].device)
            st["handle"] = kv.PagedLayers(st["k"], st["v"], table)
    return st["handle"]


def run(st):
    op = st["case"]["op"]
    if not own:
        return {"tree": _tree, "copy": _copy, "compact": _compact, "beam": _beam}[op](st)
    from expertrelay_b200 import beam, kv

    if op == "beam":
        scores, beams, tokens = beam.select(st["logits"], st["scores"], st["case"]["count"])
        return {"scores": scores, "beams": beams, "tokens": tokens}
    cache = _handle(st)
    if op == "tree":
        return {"out": kv.attend_tree(cache, st["q"], st["lens"], st["starts"], st["parents"])}
    if op == "copy":
        kv.copy_pages(cache, st["src"], st["dst"], used=st["used"])
        return {"k": st["k"], "v": st["v"]}
    lens = kv.compact(cache, st["start"], st["keep"], st["counts"])
    return {"lens": lens, "k": st["k"], "v": st["v"]}


# ---- the plain forms ---------------------------------------------------------
def _tree(st):
    case, parents = st["case"], st["parents"].long()
    kh, g, d, ps = case["kv_heads"], case["group"], case["dim"], case["page"]
    table, lens, starts = st["table"].long(), st["lens"].long(), st["starts"].long()
    trees, top, places = case["trees"], case["nodes"], table.shape[1] * ps
    dev = parents.device
    # the nodes of every tree in a row of their own, `top` wide
    at = torch.arange(top, device=dev)
    there = at[None] < (starts[1:] - starts[:-1])[:, None]                      # [trees, top]
    row = (starts[:-1, None] + at[None]).clamp(max=parents.shape[0] - 1)
    up = torch.where(there, parents[row], torch.full_like(row, -1))
    # sees[t, i, j]: j is i or one of its ancestors (the squares of "self or parent")
    sees = torch.eye(top, device=dev).expand(trees, top, top).clone()
    sees.scatter_add_(2, up.clamp(min=0)[..., None], (up >= 0).float()[..., None])
    for _ in range(max(1, top.bit_length())):
        sees = (torch.bmm(sees, sees) > 0).float()
    q = st["q"].float()[row].reshape(trees, top, kh, g, d).permute(0, 2, 1, 3, 4).reshape(trees, kh, top * g, d)
    out = torch.empty_like(q)
    pos = torch.arange(places, device=dev)
    for t in range(trees):
        pages = table[t].clamp(min=0)
        k = st["k"][pages].transpose(0, 1).reshape(kh, places, d).float()
        v = st["v"][pages].transpose(0, 1).reshape(kh, places, d).float()
        node = pos - lens[t]
        drafted = (node >= 0) & (node < top)
        mask = (pos < lens[t])[None] | (drafted[None] & (sees[t][:, node.clamp(0, top - 1)] > 0))  # [top, places]
        mask = mask & (pos < lens[t] + starts[t + 1] - starts[t])[None]
        mask = mask[:, None].expand(-1, g, -1).reshape(top * g, places)
        s = torch.matmul(q[t] * st["scale"], k.transpose(1, 2)).masked_fill(~mask, float("-inf"))
        p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38)).masked_fill(~mask, 0.0)
        total = p.sum(-1, keepdim=True)
        v = v.masked_fill((pos >= lens[t] + starts[t + 1] - starts[t])[None, :, None], 0.0)
        out[t] = torch.matmul(p / torch.where(total == 0, torch.ones_like(total), total), v)
    out = out.reshape(trees, kh, top, g, d).permute(0, 2, 1, 3, 4).reshape(trees, top, kh * g, d)
    return {"out": out[there].to(st["q"].dtype)}


def _copy(st):
    src, dst, ps = st["src"].long(), st["dst"].long(), st["case"]["page"]
    if st["used"] is None:
        for pool in (st["k"], st["v"]):
            pool[:, dst] = pool[:, src]
    else:
        live = torch.arange(ps, device=src.device)[None] < st["used"][:, None]
        at, slot = live.nonzero(as_tuple=True)
        for pool in (st["k"], st["v"]):
            pool[:, dst[at], :, slot] = pool[:, src[at], :, slot]
    return {"k": st["k"], "v": st["v"]}


def _compact(st):
    ps, table, start = st["case"]["page"], st["table"].long(), st["start"].long()
    live = torch.arange(st["keep"].shape[1], device=start.device)[None] < st["counts"][:, None]
    row, j = live.nonzero(as_tuple=True)
    a, b = start[row] + st["keep"].long()[row, j], start[row] + j
    for pool in (st["k"], st["v"]):
        pool[:, table[row, b // ps], :, b % ps] = pool[:, table[row, a // ps], :, a % ps]
    return {"lens": (start + st["counts"]).to(torch.int32), "k": st["k"], "v": st["v"]}


def _beam(st):
    # in 64 bits: candidates of different beams may lie next to each other
    case, x = st["case"], st["logits"].double()
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    value = st["scores"].double().reshape(-1, 1) + (x - (m + torch.log(torch.exp(x - m).sum(-1, keepdim=True))))
    value = torch.where(value.isnan(), float("-inf"), value).reshape(case["batch"], -1)
    best = torch.sort(value, dim=-1, descending=True, stable=True)
    at = best.indices[:, : case["count"]]
    return {"scores": best.values[:, : case["count"]].float(), "beams": (at // case["vocab"]).to(torch.int32),
            "tokens": (at % case["vocab"]).to(torch.int32)}


# ---- the definitions in 64 bits ----------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "beam":
        scores, beams, tokens = [], [], []
        for b in range(case["batch"]):
            rows = st["logits"].reshape(case["batch"], case["beams"], -1)[b].double()
            value = st["scores"][b].double()[:, None] + (rows - torch.logsumexp(rows, -1, keepdim=True))
            value = value.nan_to_num(nan=float("-inf"), posinf=float("inf"), neginf=float("-inf")).reshape(-1)
            least = torch.topk(value, case["count"]).values[-1]
            where = (value >= least).nonzero()[:, 0]
            pairs = list(zip(value[where].tolist(), where.tolist()))
            pairs = sorted(pairs, key=lambda p: (-p[0], p[1]))[: case["count"]]
            scores.append([p[0] for p in pairs])
            beams.append([p[1] // case["vocab"] for p in pairs])
            tokens.append([p[1] % case["vocab"] for p in pairs])
        return {"scores": torch.tensor(scores, dtype=torch.float64),
                "beams": torch.tensor(beams, dtype=torch.int32), "tokens": torch.tensor(tokens, dtype=torch.int32)}
    ps = case["page"]
    if case["op"] == "copy":
        k, v = st["k"].double(), st["v"].double()
        pairs = zip(st["src"].tolist(), st["dst"].tolist(), _used(case))
        for a, b, n in pairs:
            for pool in (k, v):
                pool[:, b].narrow(2, 0, n).copy_(pool[:, a].narrow(2, 0, n))
        return {"k": k, "v": v}
    if case["op"] == "compact":
        k, v = st["k"].double(), st["v"].double()
        table = st["table"].cpu()
        for s, n in enumerate(_counts(case)):
            first = int(st["start"][s])
            for pool in (k, v):
                was = torch.cat([pool[:, p] for p in table[s].tolist() if p >= 0], 2)  # [layers, heads, places, d]
                now = was.clone()
                now[:, :, first:first + n] = was[:, :, (first + st["keep"][s, :n].long())]
                for o, p in enumerate(p for p in table[s].tolist() if p >= 0):
                    pool[:, p] = now[:, :, o * ps:(o + 1) * ps]
        lens = [int(a) + n for a, n in zip(st["start"].tolist(), _counts(case))]
        return {"lens": torch.tensor(lens, dtype=torch.int32), "k": k, "v": v}
    kh, g, d = case["kv_heads"], case["group"], case["dim"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    at = 0
    for t, (n, m) in enumerate(zip(_contexts(case), _nodes(case))):
        pages = st["table"][t, : -(-(n + m) // ps)].long()
        k, v = (torch.cat(list(x[pages].double()), 1)[:, : n + m] for x in (st["k"], st["v"]))
        q = st["q"][at:at + m].double().reshape(m, kh, g, d)
        s = torch.einsum("mhgd,hnd->mhgn", q, k) / math.sqrt(d)
        path = []  # each node's ancestors and itself
        for i, p in enumerate(_parents(case, t, m)):
            path.append((path[p] if p >= 0 else []) + [i])
        hidden = torch.ones((m, m), dtype=torch.bool)
        for i, seen in enumerate(path):
            hidden[i, seen] = False
        s[..., n:] = s[..., n:].masked_fill(hidden.to(s.device)[:, None, None], float("-inf"))
        out[at:at + m] = torch.einsum("mhgn,hnd->mhgd", torch.softmax(s, -1), v).reshape(m, kh * g, d)
        at += m
    return {"out": out}
