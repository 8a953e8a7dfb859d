"""GPU: attention of trees of drafted tokens against its definition in 64 bits
(tests/tree_ref.py), at the shapes, lengths, pages and masks where it can go wrong."""

from __future__ import annotations

import numpy as np
import pytest
import torch
from kv_ref import U, attend_exact, make_cache, result_bound, result_error
from tree_ref import check_trees

from expertrelay_b200 import _lib, kv

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TYPES = [(F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)]


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _tree(rng, n, kind="tree"):
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "flat":
        return [-1] * n
    return [int(rng.integers(-1, i)) if i else -1 for i in range(n)]


def _case(seed, lens, trees, kv_heads, group, d, ps, cache_dtype, q_dtype, layout="hnd"):
    gen = torch.Generator().manual_seed(seed)
    k, v, table = make_cache(gen, [n + len(t) for n, t in zip(lens, trees)], kv_heads, d, ps, cache_dtype, layout=layout)
    rows = sum(len(t) for t in trees)
    q = torch.randn((rows, kv_heads * group, d), generator=gen).to(q_dtype).cuda()
    starts = np.concatenate([[0], np.cumsum([len(t) for t in trees])])
    parents = [p for t in trees for p in t]
    return kv.PagedKV(k, v, table), q, _i32(lens), _i32(starts.tolist()), _i32(parents)


@pytest.mark.parametrize(("cache_dtype", "q_dtype"), TYPES)
@pytest.mark.parametrize(("kv_heads", "group", "d", "ps"), [
    (16, 1, 128, 16), (4, 8, 128, 64), (2, 3, 64, 24), (3, 2, 80, 7), (1, 16, 96, 1), (2, 5, 256, 32), (1, 4, 8, 5),
    (2, 1, 192, 128), (1, 2, 136, 16), (1, 33, 64, 16),
])
def test_trees_match_the_definition(cuda, cache_dtype, q_dtype, kv_heads, group, d, ps):
    rng = np.random.default_rng(d + group)
    # empty and short contexts, ends around a tile of 32, 64 and 128 keys, drafts across a tile's and a page's end
    lens = [0, 0, 1, 31, 33, 60, 64, 100, 127, 128, 333, 1501]
    sizes = [1, 9, 3, 2, 17, 12, 1, 40, 5, 64, 8, 33]
    trees = [_tree(rng, n, kind) for n, kind in zip(sizes, ["tree", "chain", "tree", "flat"] * 3)]
    cache, q, ln, starts, parents = _case(d + group, lens, trees, kv_heads, group, d, ps, cache_dtype, q_dtype)
    out = kv.attend_tree(cache, q, ln, starts, parents)
    assert out.dtype == q_dtype and tuple(out.shape) == tuple(q.shape)
    check_trees(cache, q, lens, trees, out)
    cache.check()
    assert torch.equal(out, kv.attend_tree(cache, q, ln, starts, parents))  # bit for bit again


@pytest.mark.parametrize(("cache_dtype", "q_dtype"), TYPES)
@pytest.mark.parametrize(("length", "nodes", "kv_heads", "group", "d"), [
    (0, 256, 1, 1, 64), (5000, 1, 2, 4, 128), (640, 8, 16, 1, 128), (20001, 16, 2, 6, 64), (3000, 130, 1, 2, 128),
    (700, 256, 2, 3, 32), (1200, 70, 1, 4, 256),
])
def test_one_tree(cuda, cache_dtype, q_dtype, length, nodes, kv_heads, group, d):
    tree = _tree(np.random.default_rng(nodes), nodes)
    cache, q, ln, starts, parents = _case(length, [length], [tree], kv_heads, group, d, 16, cache_dtype, q_dtype)
    check_trees(cache, q, [length], [tree], kv.attend_tree(cache, q, ln, starts, parents))
    cache.check()


@pytest.mark.parametrize(("cache_dtype", "q_dtype"), TYPES)
def test_many_uneven_trees(cuda, cache_dtype, q_dtype):
    rng = np.random.default_rng(3)
    lens = [int(n) for n in np.exp(rng.uniform(0, 7.5, 70))]
    trees = [_tree(rng, int(n)) for n in np.exp(rng.uniform(0, 3.5, 70))]
    cache, q, ln, starts, parents = _case(9, lens, trees, 2, 2, 64, 32, cache_dtype, q_dtype)
    check_trees(cache, q, lens, trees, kv.attend_tree(cache, q, ln, starts, parents))


@pytest.mark.parametrize(("cache_dtype", "q_dtype"), TYPES)
@pytest.mark.parametrize("layout", ["nhd", "wide"])
def test_strides_scales_and_rows_of_no_tree(cuda, cache_dtype, q_dtype, layout):
    rng = np.random.default_rng(5)
    lens, trees = [200, 0, 77], [_tree(rng, 11), _tree(rng, 4), _tree(rng, 30)]
    cache, q, _, _, parents = _case(5, lens, trees, 3, 2, 64, 16, cache_dtype, q_dtype, layout=layout)
    order = [2, 0, 1]
    rows = q.shape[0]
    wide = torch.randn((rows + 7, 6 * 64 + 40), device="cuda").to(q_dtype)
    wide[3:3 + rows, 8:8 + 6 * 64] = q.reshape(rows, -1)
    qs = wide[:, 8:8 + 6 * 64].view(rows + 7, 6, 64)
    out = torch.full((rows + 7, 6, 64), 7.0, dtype=q_dtype, device="cuda")
    # the trees begin behind three rows of no tree, four follow; sequences in another order
    starts = _i32([3, 14, 18, 48])
    tables = torch.full((3, cache.width + 3), -7, dtype=torch.int32, device="cuda")
    tables[order, :cache.width] = cache.table
    other = kv.PagedKV(cache.k, cache.v, tables[:, :cache.width])
    more = torch.cat([_i32([-9, -9, 500]), parents, _i32([3, 3, 3, 3])])
    assert kv.attend_tree(other, qs, _i32(lens), starts, more, seqs=_i32(order), scale=0.3, out=out) is out
    check_trees(other, qs, lens, trees, out, first=3, seqs=order, scale=0.3)
    assert torch.all(out[:3] == 7.0) and torch.all(out[3 + rows:] == 7.0)
    other.check()


@pytest.mark.parametrize(("cache_dtype", "q_dtype"), TYPES)
def test_masked_places_change_nothing(cuda, cache_dtype, q_dtype):
    """NaN and infinite keys and values of nodes that a node does not see; scores of -inf."""
    lens, tree = [150], [-1, 0, 0, 1, 2, -1, 5]
    cache, q, ln, starts, parents = _case(7, lens, [tree], 2, 3, 64, 16, cache_dtype, q_dtype)
    want = kv.attend_tree(cache, q, ln, starts, parents)
    for node, key, value in ((5, float("nan"), float("nan")), (2, float("inf"), float("-inf")), (1, 1.0, float("inf"))):
        place = lens[0] + node
        page = int(cache.table[0, place // 16])
        was = cache.k[page, :, place % 16].clone(), cache.v[page, :, place % 16].clone()
        cache.k[page, :, place % 16], cache.v[page, :, place % 16] = key, value
        got = kv.attend_tree(cache, q, ln, starts, parents)
        blind = [i for i, p in enumerate(tree) if i != node and p != node and (p < 0 or tree[p] != node)]
        assert torch.equal(got[blind], want[blind])
        assert not torch.isfinite(got[node]).any()
        cache.k[page, :, place % 16], cache.v[page, :, place % 16] = was
    # no context, and a node whose own key scores -inf: nothing is left of the row
    cache, q, ln, starts, parents = _case(8, [0], [[-1]], 1, 1, 64, 16, cache_dtype, q_dtype)
    q.fill_(1.0)
    cache.k[int(cache.table[0, 0]), :, 0] = float("-inf")
    out = kv.attend_tree(cache, q, ln, starts, parents)
    assert torch.all(out == 0) or (cache_dtype == F32 and torch.isnan(out).all())


@pytest.mark.parametrize(("cache_dtype", "q_dtype"), TYPES)
def test_bad_trees_spoil_their_own_rows(cuda, cache_dtype, q_dtype):
    rng = np.random.default_rng(1)
    lens, trees = [300, 40, 77, 20], [_tree(rng, 6), _tree(rng, 5), _tree(rng, 7), _tree(rng, 4)]
    cache, q, ln, starts, parents = _case(11, lens, trees, 2, 2, 64, 16, cache_dtype, q_dtype)
    want = kv.attend_tree(cache, q, ln, starts, parents)
    rows = slice(6, 11)
    others = [i for i in range(22) if not 6 <= i < 11]

    def spoilt(words, cache=cache, ln=ln, parents=parents, starts=starts, seqs=None):
        got = kv.attend_tree(cache, q, ln, starts, parents, seqs=seqs)
        assert torch.isnan(got[rows]).all() and torch.equal(got[others], want[others])
        with pytest.raises(ValueError, match=words):
            cache.check()
        cache.check()

    for bad in (4, 7, -2, 2**31 - 1, -2**31):
        p = parents.clone()
        p[6 + 4] = bad
        spoilt("tree", parents=p)
    for bad in (-1, cache.width * 16, 2**31 - 1):
        n = ln.clone()
        n[1] = bad
        spoilt("length", ln=n)
    for bad in (-1, 4, 2**31 - 1):
        spoilt("sequence", seqs=_i32([0, bad, 2, 3]))
    for bad, page in ((-1, 0), (cache.num_pages, 2), (2**31 - 1, 2)):
        table = cache.table.clone()
        table[1, page] = bad
        spoilt("page", cache=kv.PagedKV(cache.k, cache.v, table))
    # rows outside the queries or descending: the tree has none, its rows are left
    for bad in ([0, 6, 5, 18, 22], [0, 6, 30, 18, 22], [0, -6, 11, 18, 22]):
        out = torch.full_like(q, 3.0)
        kv.attend_tree(cache, q, ln, _i32(bad), parents, out=out)
        assert torch.equal(out[18:], want[18:])
        with pytest.raises(ValueError, match="tree"):
            cache.check()


def test_too_many_nodes(cuda):
    tree = list(range(-1, 256))  # 257
    cache, q, ln, starts, parents = _case(2, [10], [tree], 1, 1, 64, 16, BF16, BF16)
    assert torch.isnan(kv.attend_tree(cache, q, ln, starts, parents)).all()
    with pytest.raises(ValueError, match="tree"):
        cache.check()


@pytest.mark.parametrize(("cache_dtype", "q_dtype"), TYPES)
def test_captured_calls_follow_their_tensors(cuda, cache_dtype, q_dtype):
    """One graph, replayed over other lengths, trees and tables; two graphs of one cache; another stream."""
    rng = np.random.default_rng(2)
    lens, trees = [300, 5, 700], [_tree(rng, 8) for _ in range(3)]
    cache, q, ln, starts, parents = _case(4, lens, trees, 2, 4, 128, 16, cache_dtype, q_dtype)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kv.attend_tree(cache, q, ln, starts, parents)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(kv.attend_tree(cache, q, ln, starts, parents))
        graphs.append(g)
    for lens, sizes in (([10, 705, 0], [1, 20, 3]), ([300, 5, 700], [8, 8, 8]), ([0, 0, 3], [2, 2, 2])):
        trees = [_tree(rng, n) for n in sizes]
        lens = [min(n, 13 * 16 - m if t == 1 else n) for t, (n, m) in enumerate(zip(lens, sizes))]
        lens = [min(n, (int((cache.table[t] >= 0).sum()) * 16) - m) for t, (n, m) in enumerate(zip(lens, sizes))]
        trees = [t if n >= 0 else [-1] for t, n in zip(trees, lens)]
        lens = [max(n, 0) for n in lens]
        ln.copy_(_i32(lens))
        starts.copy_(_i32(np.concatenate([[0], np.cumsum([len(t) for t in trees])]).tolist()))
        flat = [p for t in trees for p in t]
        parents[:len(flat)] = _i32(flat)
        # every slot that these lengths reach holds something
        cache.k.nan_to_num_(nan=0.25)
        cache.v.nan_to_num_(nan=0.5)
        for g, out in zip(graphs, outs):
            out.zero_()
            g.replay()
            check_trees(cache, q, lens, trees, out)
    cache.check()


def test_refusals(cuda):
    cache, q, ln, starts, parents = _case(2, [10], [[-1, 0]], 2, 2, 64, 16, BF16, BF16)
    for change, words in (({"lens": ln.long()}, "lens"), ({"lens": _i32([1, 2])}, "lens"), ({"starts": starts[:0]}, "starts"),
                          ({"starts": starts.float()}, "starts"), ({"starts": None}, "starts"), ({"parents": parents[:1]}, "parents"),
                          ({"q": q.half()}, "q:"), ({"q": q[:, :3]}, "heads"), ({"seqs": starts}, "seqs"),
                          ({"out": q[:1].clone()}, "out"),
                          ({"workspace": torch.empty(0, dtype=torch.uint8, device="cuda")}, "workspace")):
        args = {"q": q, "lens": ln, "starts": starts, "parents": parents, **change}
        with pytest.raises(ValueError, match=words):
            kv.attend_tree(cache, args.pop("q"), args.pop("lens"), args.pop("starts"), args.pop("parents"), **args)
    with pytest.raises(ValueError, match="seqs"):
        kv.attend_tree(cache, q, _i32([1, 1]), _i32([0, 1, 2]), parents)
    assert kv.attend_tree(cache, q, ln[:0], starts[:1], parents).shape == q.shape
    assert kv.attend_tree(cache, q[:0], _i32([0]), _i32([0, 0]), parents[:0]).shape == (0, 4, 64)


@pytest.mark.parametrize(("cache_dtype", "q_dtype"), TYPES)
def test_one_sequence_in_two_trees(cuda, cache_dtype, q_dtype):
    """Two trees over the same places, among others, and the same pages under other sequences: as each alone."""
    rng = np.random.default_rng(6)
    lens, trees = [150, 90], [_tree(rng, 6), _tree(rng, 6)]
    cache, q, _, _, parents = _case(6, lens, trees, 2, 2, 64, 16, cache_dtype, q_dtype)
    two = kv.PagedKV(cache.k, cache.v, torch.cat([cache.table, cache.table[:1]]))
    q3 = torch.cat([q[:6], q[6:], q[:6] * 0.5, q[:6]])
    p3 = torch.cat([parents[:6], parents[6:], parents[:6], parents[:6]])
    lens4, seqs = [150, 90, 150, 150], [0, 1, 0, 2]
    out = kv.attend_tree(two, q3, _i32(lens4), _i32([0, 6, 12, 18, 24]), p3, seqs=_i32(seqs))
    check_trees(two, q3, lens4, [trees[0], trees[1], trees[0], trees[0]], out, seqs=seqs)
    assert torch.equal(out[:6], out[18:])
    cache.check()


@pytest.mark.parametrize(("cache_dtype", "q_dtype"), TYPES)
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30, 2.0])
def test_scales(cuda, cache_dtype, q_dtype, scale):
    rng = np.random.default_rng(8)
    lens, trees = [100, 3], [_tree(rng, 9), _tree(rng, 2)]
    cache, q, ln, starts, parents = _case(8, lens, trees, 2, 3, 72, 16, cache_dtype, q_dtype)
    check_trees(cache, q, lens, trees, kv.attend_tree(cache, q, ln, starts, parents, scale=scale), scale=scale)


@pytest.mark.parametrize(("cache_dtype", "q_dtype"), TYPES)
@pytest.mark.parametrize("off", [1, 2, 4])
def test_queries_off_16_bytes(cuda, cache_dtype, q_dtype, off):
    """Rows at odd strides and addresses: only out and the cache have to lie on 16 bytes."""
    rng = np.random.default_rng(off)
    lens, trees = [70, 33], [_tree(rng, 7), _tree(rng, 12)]
    cache, q, ln, starts, parents = _case(off, lens, trees, 2, 2, 64, 16, cache_dtype, q_dtype)
    flat = torch.zeros(19 * 259 + off, dtype=q_dtype, device="cuda")
    odd = flat[off:].view(19, 259)[:, :256]
    odd.copy_(q.reshape(19, 256))
    out = kv.attend_tree(cache, odd.view(19, 4, 64), ln, starts, parents)
    assert torch.equal(out, kv.attend_tree(cache, q, ln, starts, parents))


@pytest.mark.parametrize(("cache_dtype", "q_dtype"), TYPES)
def test_a_chain_is_a_piece_of_a_text(cuda, cache_dtype, q_dtype):
    """attend over the same places, row by row: two kernels, each within its rounding of the definition."""
    lens, trees = [517], [_tree(None, 100, "chain")]
    cache, q, ln, starts, parents = _case(12, lens, trees, 2, 4, 128, 16, cache_dtype, q_dtype)
    got = kv.attend_tree(cache, q, ln, starts, parents).double()
    want = kv.attend(cache, q, _i32([518 + i for i in range(100)]), seqs=_i32([0] * 100)).double()
    # a step of the results' type, where both round, or a few of 32 bits' of the row's greatest
    step = torch.finfo(q_dtype).eps if q_dtype == BF16 else 2.0 ** -18
    assert torch.all((got - want).abs() <= step * want.abs().amax(-1, keepdim=True))


@pytest.mark.parametrize(("cache_dtype", "q_dtype"), TYPES)
@pytest.mark.parametrize(("kv_heads", "group", "n", "d", "nodes"), [
    (4, 4, 1008, 64, 16), (4, 2, 1008, 128, 60), (2, 3, 2000, 256, 20), (1, 1, 4800, 128, 1), (2, 16, 480, 96, 9), (4, 1, 20000, 64, 4),
])
@pytest.mark.parametrize("size", [1.0, 0.02])
def test_trees_are_as_exact_as_32_bits(cuda, cache_dtype, q_dtype, kv_heads, group, n, d, nodes, size):
    """size: the spread of the scores. result_bound counts d / 8 products for a score and two sums over 16 keys; here
    they are d / 16 and 64 / 16, for each pair of the operands' parts that is multiplied: 1 and 2 of bf16 queries over a
    bf16 cache, 3 and 3 of fp32 ones, 6 and 6 over an fp32 cache. Each cuts up to U of a sum that grows as it is
    added up: half of that. Weights in two parts, where the result has 8 bits, lack 2^-18 at the most."""
    score, value = (6, 6) if cache_dtype == F32 else (3, 3) if q_dtype == F32 else (1, 2)
    bound = result_bound(d, n, size) + (score * d / 32 * size + value * 4 / 2) * U
    if cache_dtype == q_dtype == BF16:
        bound += 2.0 ** -18
    gen = torch.Generator(device="cuda").manual_seed(n + d)
    trees = max(1, min(64, 3000000 // (n * d)))
    each = -(-(n + nodes) // 16)
    k, v = (torch.randn((trees * each, kv_heads, 16, d), generator=gen, device="cuda").to(cache_dtype) for _ in range(2))
    table = torch.randperm(trees * each, generator=gen, device="cuda").to(torch.int32).view(trees, each)
    cache = kv.PagedKV(k, v, table)
    seen = [x[table.long()].transpose(1, 2).reshape(trees, kv_heads, each * 16, d) for x in (k, v)]
    calls = 1 if q_dtype == F32 else max(1, min(40, 400000 // (trees * nodes * kv_heads * group * d)))
    outs, wants = [], []
    for _ in range(calls):
        q = torch.randn((trees * nodes, kv_heads * group, d), generator=gen, device="cuda").to(q_dtype)
        starts = torch.arange(trees + 1, dtype=torch.int32, device="cuda") * nodes
        outs.append(kv.attend_tree(cache, q, _i32([n] * trees), starts, _i32([-1] * (trees * nodes)), scale=size * d ** -0.5))
        of = q.view(trees, nodes, kv_heads, group, d)
        want = torch.empty(of.shape, dtype=torch.float64, device="cuda")
        for i in range(nodes):  # the context and the node's own place
            kk, vv = (torch.cat([x[:, :, :n], x[:, :, n + i:n + i + 1]], 2) for x in seen)
            want[:, i] = attend_exact(of[:, i], kk, vv, size * d ** -0.5)
        wants.append(want.view(q.shape))
    got = result_error(torch.stack(outs), torch.stack(wants), q_dtype)
    assert got <= bound, f"{got:.3g} of the result, {bound:.3g} allowed"
    cache.check()


@pytest.mark.parametrize(("cache_dtype", "d"), [(BF16, 128), (F32, 128), (F32, 256)])
def test_pools_past_32_bits(cuda, cache_dtype, d):
    """The last pages of pools of 4.3 GB each: attention, copies and places moved, as in a pool of those pages alone."""
    ps, pages = 64, 10
    rng = np.random.default_rng(4)
    lens, trees = [300, 211], [_tree(rng, 9), _tree(rng, 20)]
    gen = torch.Generator(device=cuda).manual_seed(3)
    many = (2**32 + 2**26) // (ps * d * cache_dtype.itemsize)
    big = [torch.empty((many, 1, ps, d), dtype=cache_dtype, device=cuda) for _ in range(2)]
    small = [torch.randn((pages + 1, 1, ps, d), generator=gen, device=cuda).to(cache_dtype) for _ in range(2)]
    for a, b in zip(big, small):
        a[many - pages - 1:] = b
    table = _i32(rng.permutation(pages).reshape(2, 5).tolist())
    caches = [kv.PagedKV(*small, table), kv.PagedKV(*big, table + (many - pages - 1))]
    q = torch.randn((29, 4, d), generator=gen, device=cuda).to(cache_dtype)
    args = _i32(lens), _i32([0, 9, 29]), _i32(trees[0] + trees[1])
    want, got = (kv.attend_tree(c, q, *args) for c in caches)
    assert torch.equal(want, got)
    for c, first in zip(caches, (0, many - pages - 1)):
        kv.copy_pages(c, _i32([first + 2]), _i32([first + pages]))
        kv.compact(c, _i32([250, 200]), _i32([[3, 40, 41], [0, 9, 30]]), _i32([3, 3]))
        c.check()
    for a, b in zip(big, small):
        assert torch.equal(a[many - pages - 1:], b)


@pytest.mark.parametrize(("cache_dtype", "q_dtype"), TYPES)
@pytest.mark.parametrize(("lens", "kv_heads", "d"), [([40, 3], 2, 64), ([5000], 2, 128), ([200, 700, 90], 8, 256)])
def test_a_wait_that_runs_out_is_reported_and_spoils_every_row(cuda, cache_dtype, q_dtype, lens, kv_heads, d):
    """The warps that keep the sums wait for what never comes, when their CTA's other warps are through: the call ends,
    with its rows NaN and a RuntimeError from check(); the next one is as ever."""
    rng = np.random.default_rng(3)
    trees = [_tree(rng, 5) for _ in lens]
    cache, q, ln, starts, parents = _case(13, lens, trees, kv_heads, 2, d, 16, cache_dtype, q_dtype)
    want = kv.attend_tree(cache, q, ln, starts, parents)
    out, lib = torch.full((q.shape[0] + 1, *q.shape[1:]), 7.0, dtype=q_dtype, device="cuda"), _lib.lib()
    _lib.check(lib.er_kv_tree_test_stall(1000000, 1), "er_kv_tree_test_stall")
    try:
        more = torch.cat([q, q[:1]]), torch.cat([parents, _i32([-1])])
        kv.attend_tree(cache, more[0], ln, starts, more[1], out=out)
    finally:
        _lib.check(lib.er_kv_tree_test_stall(0, 0), "er_kv_tree_test_stall")
    assert torch.isnan(out[:-1]).all() and torch.all(out[-1] == 7.0)
    with pytest.raises(RuntimeError, match="gave up"):
        cache.check()
    assert torch.equal(kv.attend_tree(cache, q, ln, starts, parents), want)
    cache.check()


def test_the_stall_of_waits_has_two_modes():
    assert _lib.lib().er_kv_tree_test_stall(0, 2) == _lib.ER_EINVAL and _lib.lib().er_kv_tree_test_stall(0, -1) == _lib.ER_EINVAL


@pytest.mark.parametrize(("cache_dtype", "q_dtype"), TYPES)
@pytest.mark.parametrize(("lens", "d"), [([700, 20, 0], 128), ([9000], 64)])
def test_results_in_the_place_of_their_queries(cuda, cache_dtype, q_dtype, lens, d):
    rng = np.random.default_rng(2)
    trees = [_tree(rng, 70) for _ in lens]
    cache, q, ln, starts, parents = _case(15, lens, trees, 2, 3, d, 16, cache_dtype, q_dtype)
    want = kv.attend_tree(cache, q, ln, starts, parents)
    assert kv.attend_tree(cache, q, ln, starts, parents, out=q) is q and torch.equal(q, want)


def test_results_over_other_queries_are_refused(cuda):
    cache, q, ln, starts, parents = _case(15, [30], [[-1, 0]], 2, 3, 256, 16, BF16, BF16)
    both = torch.empty((3, 6, 256), dtype=BF16, device="cuda")
    for queries, out in ((q, q), (both[:2], both[1:])):
        with pytest.raises(ValueError, match="share memory"):
            kv.attend_tree(cache, queries, ln, starts, parents, out=out)
    assert kv.attend_tree(cache, both[:2], ln, starts, parents, out=q) is q


@pytest.mark.parametrize(("cache_dtype", "q_dtype"), TYPES)
@pytest.mark.parametrize(("trees", "kv_heads", "group", "n", "d", "nodes"), [(4, 40, 1, 20000, 64, 3), (6, 32, 2, 8000, 128, 9), (3, 64, 4, 5000, 256, 2)])
def test_long_units_of_one_cta_are_as_exact(cuda, cache_dtype, q_dtype, trees, kv_heads, group, n, d, nodes):
    """More units than CTAs, so that one goes through a unit's hundreds of tiles by itself: the bound of
    test_trees_are_as_exact_as_32_bits."""
    score, value = (6, 6) if cache_dtype == F32 else (3, 3) if q_dtype == F32 else (1, 2)
    bound = result_bound(d, n) + (score * d / 32 + value * 4 / 2) * U
    if cache_dtype == q_dtype == BF16:
        bound += 2.0 ** -18
    gen = torch.Generator(device="cuda").manual_seed(n + d)
    each = -(-(n + nodes) // 16)
    k, v = (torch.randn((trees * each, kv_heads, 16, d), generator=gen, device="cuda").to(cache_dtype) for _ in range(2))
    table = torch.randperm(trees * each, generator=gen, device="cuda").to(torch.int32).view(trees, each)
    cache = kv.PagedKV(k, v, table)
    outs, wants = [], []
    for _ in range(1 if q_dtype == F32 else 12):  # enough of them that cross a border between two bf16 values
        q = torch.randn((trees * nodes, kv_heads * group, d), generator=gen, device="cuda").to(q_dtype)
        starts = torch.arange(trees + 1, dtype=torch.int32, device="cuda") * nodes
        outs.append(kv.attend_tree(cache, q, _i32([n] * trees), starts, _i32([-1] * (trees * nodes))))
        of = q.view(trees, nodes, kv_heads, group, d)
        want = torch.empty(of.shape, dtype=torch.float64, device="cuda")
        for t in range(trees):
            kk, vv = (x[table[t].long()].transpose(0, 1).reshape(1, kv_heads, each * 16, d) for x in (k, v))
            for i in range(nodes):
                see = [torch.cat([x[:, :, :n], x[:, :, n + i:n + i + 1]], 2) for x in (kk, vv)]
                want[t, i] = attend_exact(of[t, i][None], *see, d ** -0.5)[0]
        wants.append(want.view(q.shape))
    got = result_error(torch.stack(outs), torch.stack(wants), q_dtype)
    assert got <= bound, f"{got:.3g} of the result, {bound:.3g} allowed"
    cache.check()
