"""GPU: the paged key-value cache's operators against their definitions in
64 bits (tests/kv_ref.py), at the lengths, pages, strides and masks where
they can go wrong."""

from __future__ import annotations

import numpy as np
import pytest
import torch
from kv_ref import attend_row, attend_tolerance, bounds_of, choose, half_step, make_cache, page_scores, tokens

from expertrelay_b200 import kv

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _i32(x, device="cuda"):
    return torch.tensor(x, dtype=torch.int32, device=device)


def _case(seed, lens, kv_heads, group, d, ps, cache_dtype, q_dtype, layout="hnd", rows=None):
    gen = torch.Generator().manual_seed(seed)
    k, v, table = make_cache(gen, lens, kv_heads, d, ps, cache_dtype, layout=layout)
    q = torch.randn((len(lens) if rows is None else rows, kv_heads * group, d), generator=gen).to(q_dtype).cuda()
    return kv.PagedKV(k, v, table), q


def _check_attend(cache, q, lens, out, *, seqs=None, scale=None, mass=None, mass0=None, picks=None):
    d = cache.head_dim
    scale = d ** -0.5 if scale is None else scale
    table = cache.table.cpu()
    for r, n in enumerate(lens):
        s = r if seqs is None else seqs[r]
        kk, vv = tokens(cache.k, table, s, n), tokens(cache.v, table, s, n)
        want, weight, spread, size = attend_row(q[r].double().cpu().numpy(), kk, vv, scale,
                                                None if picks is None else picks[r])
        tol = attend_tolerance(want, spread, size, d, n, out.dtype)
        got = out[r].double().cpu().numpy()
        assert np.all(np.abs(got - want) <= tol), \
            f"row {r} of {n}: off by {np.max(np.abs(got - want) / tol):.3g} of the tolerance"
        if mass is not None:
            grown = mass[r, :, :n].double().cpu().numpy() - mass0[r, :, :n].double().cpu().numpy()
            eps = 2 * (d + 4) * 2.0 ** -23 * size + (2 * n + 16) * 2.0 ** -23
            slack = eps * weight + half_step(F32) * np.abs(mass[r, :, :n].double().cpu().numpy()) + 1e-30
            assert np.all(np.abs(grown - weight) <= slack), f"mass of row {r}"
            assert torch.equal(mass[r, :, n:], mass0[r, :, n:])


@pytest.mark.parametrize(("cache_dtype", "q_dtype"), [(F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize(("kv_heads", "group", "d", "ps"), [
    (16, 1, 128, 16), (4, 8, 128, 64), (2, 3, 64, 24), (3, 2, 80, 7), (1, 16, 96, 1), (2, 5, 256, 32), (1, 4, 8, 5),
    (2, 1, 192, 128), (1, 33, 64, 16),
])
def test_attend_matches_the_definition(cuda, cache_dtype, q_dtype, kv_heads, group, d, ps):
    # empty, one, around a chunk of 16 keys, around a tile, a page's end inside a tile, odd and long
    lens = [0, 1, 15, 16, 17, 63, 64, 65, 129, 333, 1501]
    cache, q = _case(d + group, lens, kv_heads, group, d, ps, cache_dtype, q_dtype)
    out = kv.attend(cache, q, _i32(lens))
    assert out.dtype == q_dtype and tuple(out.shape) == tuple(q.shape)
    assert torch.all(out[0] == 0)
    _check_attend(cache, q, lens, out)
    cache.check()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("length", [1, 2, 31, 640, 5000, 40001])
def test_attend_one_row(cuda, dtype, length):
    cache, q = _case(length, [length], 2, 4, 128, 16, dtype, dtype)
    out = kv.attend(cache, q, _i32([length]))
    _check_attend(cache, q, [length], out)
    assert torch.equal(out, kv.attend(cache, q, _i32([length])))  # bit for bit again


@pytest.mark.parametrize(("cache_dtype", "q_dtype"), [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize(("rows", "kv_heads", "group", "d", "ps"), [(1, 16, 1, 128, 16), (3, 2, 5, 80, 7), (2, 1, 12, 256, 32)])
def test_attend_few_units(cuda, cache_dtype, q_dtype, rows, kv_heads, group, d, ps):
    """Few (row, key head) units, a cluster each, and the same with a table too wide for that."""
    for lens in ([577, 0, 1][:rows], [1, 130, 64][:rows], [0, 0, 0][:rows]):
        cache, q = _case(sum(lens), lens, kv_heads, group, d, ps, cache_dtype, q_dtype)
        mass = torch.rand((rows, kv_heads, 600), device="cuda")
        mass0 = mass.clone()
        out = kv.attend(cache, q, _i32(lens), mass=mass)
        _check_attend(cache, q, lens, out, mass=mass, mass0=mass0)
        wide = torch.full((rows, 40000), -1, dtype=torch.int32, device="cuda")
        wide[:, :cache.width] = cache.table
        _check_attend(cache, q, lens, kv.attend(kv.PagedKV(cache.k, cache.v, wide), q, _i32(lens)))
        cache.check()
    table = cache.table.clone()
    if rows > 1:
        lens = [5, 6, 7][:rows]
        cache, q = _case(3, lens, kv_heads, group, d, ps, cache_dtype, q_dtype)
        table = cache.table.clone()
        table[1, 0] = -9
        out = kv.attend(kv.PagedKV(cache.k, cache.v, table), q, _i32(lens))
        assert torch.isnan(out[1]).all() and not torch.isnan(out[0]).any()
        assert torch.isnan(kv.attend(cache, q, _i32([5, -1, 7][:rows]))[1]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout", ["nhd", "wide"])
def test_attend_strides(cuda, dtype, layout):
    lens = [200, 0, 77, 1]
    cache, q = _case(5, lens, 3, 2, 64, 16, dtype, dtype, layout=layout)
    wide = torch.randn((4, 6 * 64 + 40)).to(dtype).cuda()
    wide[:, 8:8 + 6 * 64] = q.reshape(4, -1)
    qs = wide[:, 8:8 + 6 * 64].view(4, 6, 64)
    assert not qs.is_contiguous()
    _check_attend(cache, q, lens, kv.attend(cache, qs, _i32(lens)))
    # a table whose rows lie apart, a scale of one's own, an output given
    table = torch.full((4, cache.width + 3), -7, dtype=torch.int32, device="cuda")
    table[:, :cache.width] = cache.table
    other = kv.PagedKV(cache.k, cache.v, table[:, :cache.width])
    out = torch.empty_like(q)
    assert kv.attend(other, qs, _i32(lens), scale=0.3, out=out) is out
    _check_attend(cache, q, lens, out, scale=0.3)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attend_rows_of_one_sequence(cuda, dtype):
    """A prompt's tokens as rows that share their sequence, in any order."""
    lens = [150, 90]
    seqs = [0] * 150 + [1, 0, 1]
    rows = list(range(1, 151)) + [90, 3, 41]
    cache, q = _case(6, lens, 2, 2, 64, 16, dtype, dtype, rows=len(rows))
    out = kv.attend(cache, q, _i32(rows), seqs=_i32(seqs))
    _check_attend(cache, q, rows, out, seqs=seqs)


def test_attend_more_rows_than_a_launch_takes(cuda):
    """More than 4096 rows go in several launches."""
    lens = [33, 70]
    cache, _ = _case(7, lens, 1, 2, 32, 16, F32, F32)
    rows = 4100
    q = torch.randn((rows, 2, 32), device="cuda")
    seqs = torch.arange(rows, device="cuda", dtype=torch.int32) % 2
    ns = (torch.arange(rows, device="cuda", dtype=torch.int32) * 7) % 34
    mass = torch.zeros((rows, 1, 40), device="cuda")
    out = kv.attend(cache, q, ns, seqs=seqs, mass=mass)
    at = [0, 1, 2, 4094, 4095, 4096, 4097, 4099]
    _check_attend(cache, q[at], ns[at].tolist(), out[at], seqs=seqs[at].tolist(), mass=mass[at],
                  mass0=torch.zeros_like(mass[at]))


@pytest.mark.parametrize(("cache_dtype", "q_dtype"), [(F32, F32), (BF16, BF16)])
@pytest.mark.parametrize("group", [1, 3, 8, 12])
def test_attend_accumulates_mass(cuda, cache_dtype, q_dtype, group):
    lens = [300, 0, 1, 64, 2049]
    cache, q = _case(group, lens, 2, group, 64, 16, cache_dtype, q_dtype)
    mass = torch.rand((5, 2, 2100), device="cuda")[:, :, :2060]  # rows apart
    mass0 = mass.clone()
    out = kv.attend(cache, q, _i32(lens), mass=mass)
    _check_attend(cache, q, lens, out, mass=mass, mass0=mass0)
    assert torch.equal(out, kv.attend(cache, q, _i32(lens)))  # the same with and without


def test_attend_infinite_scores(cuda):
    """-inf scores weigh nothing, a row of them alone is a row without keys; +inf and NaN come out as NaN."""
    for dtype in (F32, BF16):
        cache, q = _case(8, [40, 40, 40, 40], 1, 1, 64, 16, dtype, dtype)
        big = torch.finfo(dtype).max
        q[:] = 1.0
        for r, at in ((0, list(range(40))), (1, list(range(20))), (2, [30]), (3, [5])):
            for t in at:
                cache.k[int(cache.table[r, t // 16]), 0, t % 16] = {0: -big, 1: -big, 2: big, 3: float("nan")}[r]
        out = kv.attend(cache, q, _i32([40] * 4)).float()
        assert torch.all(out[0] == 0)
        v = torch.from_numpy(tokens(cache.v, cache.table, 1, 40))
        k = torch.from_numpy(tokens(cache.k, cache.table, 1, 40))
        p = torch.softmax(k[0, 20:].sum(-1) / 8, 0)
        want = p @ v[0, 20:]
        spread = (p @ v[0, 20:].abs()).numpy()
        tol = attend_tolerance(want.numpy(), spread, float(k[0, 20:].abs().sum(-1).max() / 8), 64, 40, dtype)
        assert np.all(np.abs(out[1, 0].double().cpu().numpy() - want.numpy()) <= tol)
        assert torch.isnan(out[2]).all() and torch.isnan(out[3]).all()


def test_attend_bad_pages_and_lengths_spoil_their_rows_alone(cuda):
    for dtype in (F32, BF16):
        lens = [200, 200, 200, 200, 200, 200]
        cache, q = _case(9, lens, 2, 2, 64, 16, dtype, dtype)
        table = cache.table.clone()
        table[1, 5] = cache.num_pages
        table[2, 0] = -1
        cache = kv.PagedKV(cache.k, cache.v, table)
        given = [200, 200, 200, -3, cache.width * 16 + 1, 190]
        out = kv.attend(cache, q, _i32(given))
        for r in (1, 2, 3, 4):
            assert torch.isnan(out[r]).all(), r
        for r in (0, 5):
            _check_attend(cache, q[r:r + 1], [given[r]], out[r:r + 1], seqs=[r])
        with pytest.raises(ValueError, match="page id outside the pool, a length"):
            cache.check()
        cache.check()
        out = kv.attend(cache, q, _i32([200] * 6), seqs=_i32([0, 6, -1, 0, 0, 0]))
        assert torch.isnan(out[1:3]).all() and not torch.isnan(out[[0, 3, 4, 5]]).any()
        with pytest.raises(ValueError, match="sequence outside the table"):
            cache.check()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attend_over_page_lists(cuda, dtype):
    lens = [500, 31, 0, 64]
    cache, q = _case(10, lens, 2, 3, 64, 16, dtype, dtype)
    lists = {(0, 0): [0, 4, 31], (0, 1): [31], (1, 0): [0, 1], (1, 1): [], (2, 0): [], (2, 1): [], (3, 0): [3, 1], (3, 1): [2]}
    pages, counts = torch.full((4, 2, 5), -1, dtype=torch.int32), torch.zeros((4, 2), dtype=torch.int32)
    picks = [[None, None] for _ in lens]
    for (r, h), ids in lists.items():
        pages[r, h, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
        counts[r, h] = len(ids)
        picks[r][h] = [t for p in ids for t in range(p * 16, min(lens[r], p * 16 + 16))]
    out = kv.attend(cache, q, _i32(lens), pages=pages.cuda(), counts=counts.cuda())
    _check_attend(cache, q, lens, out, picks=picks)
    cache.check()
    # an ordinal outside the table, a count outside the list: those key heads alone are spoilt
    pages[0, 0, 1], counts[3, 1] = cache.width, 6
    out = kv.attend(cache, q, _i32(lens), pages=pages.cuda(), counts=counts.cuda())
    assert torch.isnan(out[0, :3]).all() and torch.isnan(out[3, 3:]).all()
    _check_attend(cache, q[1:3], lens[1:3], out[1:3], seqs=[1, 2], picks=picks[1:3])
    assert not torch.isnan(out[0, 3:]).any() and not torch.isnan(out[3, :3]).any()


def test_attend_offsets_past_32_bits(cuda):
    """A pool whose later pages lie more than 2^32 bytes in."""
    pages, ps, d = 70000, 128, 128  # 2.3 GB a pool of one key head in bf16: byte offsets past 2^31
    k = torch.empty((pages, 2, ps, d), dtype=BF16, device="cuda")
    v = torch.empty_like(k)
    assert k.numel() * 2 > 2 ** 32
    ids = [pages - 1, 0, pages - 2, 65536]
    gen = torch.Generator().manual_seed(1)
    for p in ids:
        k[p] = torch.randn((2, ps, d), generator=gen).to(BF16).cuda()
        v[p] = torch.randn((2, ps, d), generator=gen).to(BF16).cuda()
    cache = kv.PagedKV(k, v, _i32([ids]))
    q = torch.randn((1, 4, d), generator=gen).to(BF16).cuda()
    _check_attend(cache, q, [500], kv.attend(cache, q, _i32([500])))


@pytest.mark.parametrize("cache_dtype", [F32, BF16])
@pytest.mark.parametrize(("q_dtype", "heads", "kv_heads", "d", "ps"), [
    (F32, 16, 16, 128, 16), (BF16, 8, 2, 64, 24), (F32, 3, 1, 80, 1), (BF16, 2, 2, 256, 64), (F32, 1, 1, 8, 3),
])
def test_append(cuda, cache_dtype, q_dtype, heads, kv_heads, d, ps):
    gen = torch.Generator().manual_seed(d)
    lens = [100, 9, 40]
    k, v, table = make_cache(gen, lens, kv_heads, d, ps, cache_dtype)
    cache = kv.PagedKV(k, v, table)
    seqs = [0, 1, 0, 2, 0]
    pos = [99, 0, 50, 39, 51]
    theta = 10000.0
    wide = torch.randn((5, (heads + 2 * kv_heads) * d + 24), generator=gen).to(q_dtype).cuda()
    qkv = wide[:, : (heads + 2 * kv_heads) * d]
    k0, v0 = k.clone(), v.clone()
    q = kv.append(cache, qkv, _i32(pos), heads, theta, seqs=_i32(seqs))
    assert q.dtype == q_dtype
    x = qkv.double().cpu().numpy().reshape(5, heads + 2 * kv_heads, d)
    ang = np.array(pos)[:, None] * theta ** (-2.0 * np.arange(d // 2) / d)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    a, b = x[..., :d // 2], x[..., d // 2:]
    turned = np.concatenate([a * c - b * s, b * c + a * s], -1)
    size = np.concatenate([np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)], -1)
    # cos, sin, product and sum are rounded to 32 bits, then the result to its type
    def near(got, want, by, dtype):
        assert np.all(np.abs(got - want) <= 3.01 * 2.0 ** -24 * by + half_step(dtype) * (np.abs(want) + 3.01 * 2.0 ** -24 * by) * (dtype != F32))
    near(q.double().cpu().numpy(), turned[:, :heads], size[:, :heads], q_dtype)
    for i in range(5):
        page, slot = int(table[seqs[i], pos[i] // ps]), pos[i] % ps
        near(k[page, :, slot].double().cpu().numpy(), turned[i, heads:heads + kv_heads], size[i, heads:heads + kv_heads],
             cache_dtype)
        assert torch.equal(v[page, :, slot], qkv[i].reshape(-1, d)[heads + kv_heads:].to(cache_dtype))
        k0[page, :, slot], v0[page, :, slot] = k[page, :, slot], v[page, :, slot]
    assert torch.equal(k.nan_to_num(7), k0.nan_to_num(7)) and torch.equal(v.nan_to_num(7), v0.nan_to_num(7))
    cache.check()


def test_append_far_positions_and_other_q_type(cuda):
    """Angles of far positions, where a 32-bit product would lose them."""
    k = torch.zeros((1, 1, 1, 64), dtype=F32, device="cuda")
    cache = kv.PagedKV(k, k.clone(), torch.zeros((1, 2_000_000), dtype=torch.int32, device="cuda"))
    x = torch.randn((1, 3 * 64), device="cuda")
    q = kv.append(cache, x, _i32([1_999_999]), 1, 1e6, q_dtype=BF16)
    ang = 1_999_999 * 1e6 ** (-2.0 * np.arange(32) / 64)
    a, b = x[0, 64:96].double().cpu().numpy(), x[0, 96:128].double().cpu().numpy()
    want = np.concatenate([a * np.cos(ang) - b * np.sin(ang), b * np.cos(ang) + a * np.sin(ang)])
    size = np.abs(np.concatenate([a, b])) + np.abs(np.concatenate([b, a]))
    assert np.all(np.abs(k[0, 0, 0].double().cpu().numpy() - want) <= 3.01 * 2.0 ** -24 * size)
    assert q.dtype == BF16


def test_append_leaves_bad_rows_unwritten(cuda):
    gen = torch.Generator().manual_seed(3)
    k, v, table = make_cache(gen, [32, 32], 1, 64, 16, F32)
    table[1, 1] = 99
    cache = kv.PagedKV(k, v, table)
    k0 = k.clone()
    kv.append(cache, torch.randn((5, 3 * 64), device="cuda"), _i32([32, -1, 16, 0, 0]), 1, 1e4, seqs=_i32([0, 0, 1, 2, -1]))
    assert torch.equal(k.nan_to_num(7), k0.nan_to_num(7))
    with pytest.raises(ValueError, match="page id outside the pool, a length.*, a sequence"):
        cache.check()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize(("d", "ps"), [(128, 16), (64, 24), (80, 5), (256, 64), (8, 1)])
def test_page_bounds(cuda, dtype, d, ps):
    gen = torch.Generator().manual_seed(d)
    lens, start = [100, 0, 33, 7], [0, 0, 32, 7]
    k, v, table = make_cache(gen, lens, 2, d, ps, dtype)
    k[int(table[0, 0])] = 0  # a page of zeros: codes and scale 0
    cache = kv.PagedKV(k, v, table)
    bounds = kv.PageBounds.new(cache)
    bounds.codes.fill_(11)
    bounds.scales.fill_(-1)
    kv.page_bounds(cache, bounds, _i32(lens), _i32(start))
    cache.check()
    touched = set()
    for s, n in enumerate(lens):
        if start[s] >= n:
            continue
        for o in range(start[s] // ps, -(-n // ps)):
            page = int(table[s, o])
            for h in range(2):
                lo, hi, scale = bounds_of(k[page, h, : min(ps, n - o * ps)].float().cpu().numpy())
                assert bounds.scales[page, h].item() == scale
                assert np.array_equal(bounds.codes[page, h, 0].cpu().numpy(), lo)
                assert np.array_equal(bounds.codes[page, h, 1].cpu().numpy(), hi)
                touched.add(page)
    rest = [p for p in range(cache.num_pages) if p not in touched]
    assert torch.all(bounds.codes[rest] == 11) and torch.all(bounds.scales[rest] == -1)


def _select_case(seed, lens, kv_heads, group, d, ps, dtype):
    cache, q = _case(seed, lens, kv_heads, group, d, ps, dtype, dtype)
    bounds = kv.PageBounds.new(cache)
    kv.page_bounds(cache, bounds, _i32(lens), _i32([0] * len(lens)))
    return cache, q, bounds


def _want_pages(cache, bounds, q, lens, budget, sinks, recent):
    want = []
    table, group = cache.table.cpu(), q.shape[1] // cache.kv_heads
    codes, scales = bounds.codes.cpu().numpy(), bounds.scales.cpu().numpy()
    for r, n in enumerate(lens):
        ids = table[r, : -(-n // cache.page_size)].numpy()
        row = []
        for h in range(cache.kv_heads):
            sc = page_scores(q[r, h * group:(h + 1) * group].float().cpu().numpy(), codes[ids, h, 0], codes[ids, h, 1],
                             scales[ids, h]) if len(ids) else np.zeros(0)
            row.append(choose(sc, len(ids), budget, sinks, recent))
        want.append(row)
    return want


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize(("group", "d", "ps", "budget", "sinks", "recent"), [
    (1, 128, 16, 8, 1, 2), (8, 64, 4, 64, 0, 0), (3, 80, 1, 33, 2, 3), (2, 256, 16, 1, 0, 1), (5, 8, 2, 5, 2, 3),
])
def test_select_pages(cuda, dtype, group, d, ps, budget, sinks, recent):
    lens = [1500, 0, 1, 16 * 8, 700, 333]
    cache, q, bounds = _select_case(group, lens, 2, group, d, ps, dtype)
    pages, counts = kv.select_pages(cache, bounds, q, _i32(lens), budget, sinks=sinks, recent=recent)
    cache.check()
    for r, row in enumerate(_want_pages(cache, bounds, q, lens, budget, sinks, recent)):
        for h, ids in enumerate(row):
            assert counts[r, h].item() == len(ids)
            assert pages[r, h].tolist() == ids + [-1] * (budget - len(ids)), (r, h)
    out = kv.attend(cache, q, _i32(lens), pages=pages, counts=counts)
    picks = [[[t for p in ids for t in range(p * ps, min(n, (p + 1) * ps))] for ids in row]
             for n, row in zip(lens, _want_pages(cache, bounds, q, lens, budget, sinks, recent))]
    _check_attend(cache, q, lens, out, picks=picks)


def test_select_from_a_table_too_wide_for_shared_memory(cuda):
    lens = [1500, 0, 60000]
    cache, q, bounds = _select_case(3, lens, 1, 2, 32, 1, F32)
    pages, counts = kv.select_pages(cache, bounds, q, _i32(lens), 70, sinks=2, recent=3)
    for r, (ids,) in enumerate(_want_pages(cache, bounds, q, lens, 70, 2, 3)):
        assert pages[r, 0].tolist() == ids + [-1] * (70 - len(ids)) and counts[r, 0].item() == len(ids)
    lens = [1000, 1500, 7]  # many units: one CTA each
    cache, q, bounds = _select_case(4, lens, 16, 2, 64, 4, BF16)
    pages, counts = kv.select_pages(cache, bounds, q, _i32(lens), 40, sinks=1, recent=1)
    for r, row in enumerate(_want_pages(cache, bounds, q, lens, 40, 1, 1)):
        for h, ids in enumerate(row):
            assert pages[r, h].tolist() == ids + [-1] * (40 - len(ids)) and counts[r, h].item() == len(ids)


def test_evict_more_than_shared_memory_holds(cuda):
    gen = torch.Generator().manual_seed(9)
    n, budget = 70000, 50
    k = torch.randn((n // 100, 1, 100, 8), generator=gen).cuda()
    cache = kv.PagedKV(k, k.clone(), torch.arange(n // 100, dtype=torch.int32, device="cuda")[None])
    to = kv.PagedKV(torch.zeros((1, 1, 50, 8), device="cuda"), torch.zeros((1, 1, 50, 8), device="cuda"), _i32([[0]]))
    mass = torch.randint(0, 20, (1, 1, n), generator=gen).float()
    kept, new = kv.evict(cache, _i32([n]), mass.cuda(), to, torch.zeros((1, 1, 50), device="cuda"), budget, sinks=3, recent=7)
    ids = choose(mass[0, 0].numpy(), n, budget, 3, 7)
    assert kept[0, 0].tolist() == ids and new.tolist() == [budget]
    assert torch.equal(to.k[0, 0], k.reshape(-1, 8)[ids])


@pytest.mark.parametrize(("seqs", "n", "budget"), [(38, 32768 + 100, 50), (38, 32768 + 100, 32800), (1, 8 * 32768 + 800, 270)])
def test_evict_equal_weights_fill_a_round(cuda, seqs, n, budget):
    # a round of a CTA's scan is 32768 positions, here all of them ties: by a CTA alone, and by a cluster together
    k = torch.randn((n // 4 + 1, 1, 4, 8), generator=torch.Generator().manual_seed(3)).cuda()
    table = torch.arange(n // 4 + 1, dtype=torch.int32, device="cuda").expand(seqs, -1)  # all read the same pages
    cache = kv.PagedKV(k, k, table)
    tk = torch.zeros((seqs, 1, budget, 8), device="cuda")
    to = kv.PagedKV(tk, tk.clone(), torch.arange(seqs, dtype=torch.int32, device="cuda")[:, None])
    mass = torch.full((seqs, 1, n), 0.25, device="cuda")
    mass[:, :, n - 10] = 1.0
    kept, new = kv.evict(cache, _i32([n] * seqs), mass, to, torch.zeros((seqs, 1, budget), device="cuda"), budget, sinks=0, recent=0)
    want = torch.tensor([*range(budget - 1), n - 10], dtype=torch.int32, device="cuda")
    assert torch.all(kept == want) and torch.all(new == budget)
    assert torch.equal(to.k, k.view(-1, 8)[want.long()].expand(seqs, 1, -1, -1))
    cache.check()


def test_select_ties_zeros_and_bad_rows(cuda):
    lens = [640, 640, 640, 640]
    cache, q, bounds = _select_case(4, lens, 1, 2, 64, 16, F32)
    bounds.codes[:] = 5  # every page alike: the lowest win
    bounds.scales[:] = 1.0
    q[1] = 0
    q[2, 1, 3] = float("nan")  # no page ranks
    given = [640, 640, 640, cache.width * 16 + 1]
    pages, counts = kv.select_pages(cache, bounds, q, _i32(given), 6, sinks=1, recent=1)
    for r in range(3):
        assert pages[r, 0].tolist() == [0, 1, 2, 3, 4, 39]
    assert counts[3, 0].item() == 0 and pages[3, 0].tolist() == [-1] * 6
    with pytest.raises(ValueError, match="length"):
        cache.check()
    # a bad page id is never followed, and ranks last
    table = cache.table.clone()
    table[0, 1] = -5
    cache = kv.PagedKV(cache.k, cache.v, table)
    pages, _ = kv.select_pages(cache, bounds, q, _i32([640] * 4), 6, sinks=1, recent=1)
    assert pages[0, 0].tolist() == [0, 2, 3, 4, 5, 39]
    with pytest.raises(ValueError, match="page id"):
        cache.check()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize(("d", "ps", "to_ps", "budget", "sinks", "recent"), [
    (128, 16, 16, 100, 4, 20), (64, 24, 16, 1, 0, 0), (80, 5, 7, 300, 0, 300), (256, 64, 32, 513, 4, 0), (8, 1, 3, 64, 64, 0),
])
def test_evict(cuda, dtype, d, ps, to_ps, budget, sinks, recent):
    gen = torch.Generator().manual_seed(d)
    lens = [1200, 0, 1, budget, budget + 1, 777]
    k, v, table = make_cache(gen, lens, 2, d, ps, dtype)
    cache = kv.PagedKV(k, v, table)
    width = -(-budget // to_ps)
    tk, tv = (torch.full((6 * width, 2, to_ps, d), 9.0, dtype=dtype, device="cuda") for _ in range(2))
    to = kv.PagedKV(tk, tv, torch.randperm(6 * width, generator=gen).to(torch.int32).reshape(6, width).cuda())
    mass = torch.rand((6, 2, 1250), generator=gen)
    mass = torch.where(mass < 0.4, torch.zeros(()), mass ** 3)  # many exact ties
    mass[0, 0, 100:110] = float("nan")
    mass[0, 1, 100:110] = float("inf")
    mass[5, 0, 50] = -0.0
    mass = mass.cuda()
    to_mass = torch.full((6, 2, width * to_ps), -3.0, device="cuda")
    kept, new = kv.evict(cache, _i32(lens), mass, to, to_mass, budget, sinks=sinks, recent=recent)
    cache.check()
    assert new.tolist() == [min(n, budget) for n in lens]
    host = mass.cpu().numpy()
    for s, n in enumerate(lens):
        kk, vv = tokens(k, table, s, n), tokens(v, table, s, n)
        m = min(n, budget)
        for h in range(2):
            ids = choose(host[s, h], n, budget, sinks, recent)
            assert kept[s, h].tolist() == ids + [-1] * (budget - m), (s, h)
            got_k = np.concatenate([tk[int(p), h].double().cpu().numpy() for p in to.table[s]])
            got_v = np.concatenate([tv[int(p), h].double().cpu().numpy() for p in to.table[s]])
            assert np.array_equal(got_k[:m], kk[h][ids]) and np.array_equal(got_v[:m], vv[h][ids])
            assert np.all(got_k[m:] == 9) and np.all(got_v[m:] == 9)  # behind them as it was
            assert np.array_equal(to_mass[s, h, :m].cpu().numpy(), host[s, h][ids], equal_nan=True)
            assert torch.all(to_mass[s, h, m:] == -3)


def test_evict_bad_lengths_and_pages(cuda):
    gen = torch.Generator().manual_seed(2)
    lens = [64, 64, 64]
    k, v, table = make_cache(gen, lens, 1, 64, 16, F32)
    table[2, 3] = 1000
    cache = kv.PagedKV(k, v, table)
    tk = torch.zeros((6, 1, 16, 64), device="cuda")
    to = kv.PagedKV(tk, tk.clone(), torch.arange(6, dtype=torch.int32, device="cuda").reshape(3, 2))
    mass, to_mass = torch.rand((3, 1, 64), device="cuda"), torch.zeros((3, 1, 32), device="cuda")
    kept, new = kv.evict(cache, _i32([64, 65, 64]), mass, to, to_mass, 32, sinks=0, recent=32)
    assert new.tolist() == [32, 0, 32] and kept[1, 0].tolist() == [-1] * 32
    assert kept[2, 0].tolist() == list(range(32, 64))
    assert torch.equal(tk[5], torch.zeros_like(tk[5])) and not torch.equal(tk[4], torch.zeros_like(tk[4]))
    with pytest.raises(ValueError, match="page id outside the pool, a length"):
        cache.check()


def test_refusals(cuda):
    cache, q = _case(1, [64, 64], 2, 2, 64, 16, F32, F32)
    lens = _i32([64, 64])
    bad = [
        (lambda: kv.PagedKV(cache.k.double(), cache.v.double(), cache.table), "float32 or bfloat16"),
        (lambda: kv.PagedKV(cache.k.cpu(), cache.v.cpu(), cache.table.cpu()), "CUDA tensor"),
        (lambda: kv.PagedKV(cache.k, cache.v.to(BF16), cache.table), "v: expected"),
        (lambda: kv.PagedKV(cache.k, cache.v.transpose(1, 2).contiguous().transpose(1, 2), cache.table), "strides"),
        (lambda: kv.PagedKV(cache.k, cache.v, cache.table.long()), "table"),
        (lambda: kv.PagedKV(cache.k, cache.v, cache.table.t()), "contiguous rows"),
        (lambda: kv.attend(cache, q[:, :3], lens), "3 heads over 2"),
        (lambda: kv.attend(cache, q.half(), lens), "q: expected"),
        (lambda: kv.attend(cache, q[..., :32], lens), "q: expected"),
        (lambda: kv.attend(cache, q.transpose(0, 1).contiguous().transpose(0, 1), lens), "strides"),
        (lambda: kv.attend(cache, q, lens.long()), "lens"),
        (lambda: kv.attend(cache, q, lens[:1]), "lens"),
        (lambda: kv.attend(cache, torch.cat([q, q]), _i32([1] * 4)), "4 rows over 2 sequences"),
        (lambda: kv.attend(cache, q, lens, out=q[:1]), "out"),
        (lambda: kv.attend(cache, q, lens, pages=_i32([[[0], [0]]] * 2)), "together"),
        (lambda: kv.attend(cache, q, lens, mass=torch.zeros((2, 1, 64), device="cuda")), "mass"),
        (lambda: kv.attend(cache, q, lens, mass=torch.zeros((1, 2, 64), device="cuda").expand(2, 2, 64)), "share memory"),
        (lambda: kv.append(kv.PagedKV(cache.k[:1].expand(9, -1, -1, -1), cache.v[:1].expand(9, -1, -1, -1), cache.table),
                           torch.zeros((2, 512), device="cuda"), lens, 4, 1e4), "share memory"),
        (lambda: kv.append(cache, torch.zeros((2, 512), device="cuda"), lens.long(), 4, 1e4), "positions"),
        (lambda: kv.attend(cache, q, lens, pages=_i32([[[0], [0]]] * 2), counts=_i32([[1, 1]] * 2),
                           mass=torch.zeros((2, 2, 64), device="cuda")), "not accumulated"),
        (lambda: kv.attend(cache, q, lens, mass=torch.zeros((2, 2, 64), device="cuda"),
                           workspace=torch.empty(16, dtype=torch.uint8, device="cuda")), "workspace"),
        (lambda: kv.append(cache, torch.zeros((2, 64), device="cuda"), lens, 4, 1e4), "qkv"),
        (lambda: kv.append(cache, torch.zeros((2, 512), device="cuda"), lens, 4, 0.0), "theta"),
        (lambda: kv.append(cache, torch.zeros((2, 512), device="cuda"), lens, 4, 1e4, q_dtype=torch.half), "q_dtype"),
        (lambda: kv.select_pages(cache, kv.PageBounds.new(cache), q, lens, 2, sinks=2, recent=1), "budget"),
        (lambda: kv.select_pages(cache, kv.PageBounds(torch.zeros((1, 2, 2, 64), dtype=torch.int8, device="cuda"),
                                                      torch.zeros((1, 2), device="cuda")), q, lens, 2), "not this cache's"),
        (lambda: kv.evict(cache, lens, torch.zeros((2, 2, 64), device="cuda"), cache,
                          torch.zeros((2, 2, 64), device="cuda"), 8, recent=2), "own pages"),
    ]
    for call, words in bad:
        with pytest.raises(ValueError, match=words):
            call()
    mass = torch.zeros((2, 2, 64), device="cuda")
    to = kv.PagedKV(torch.zeros_like(cache.k), torch.zeros_like(cache.v), cache.table.clone())
    with pytest.raises(ValueError, match="to_mass"):
        kv.evict(cache, lens, mass, to, mass, 8, recent=2)
    with pytest.raises(ValueError, match="share memory with mass"):
        kv.evict(cache, lens, mass[:, :, :32], to, mass[:, :, 16:], 8, recent=2)
    with pytest.raises(ValueError, match="out must be 16-byte"):
        kv.attend(cache, q, lens, out=torch.zeros(q.numel() + 1, device="cuda")[1:].view(q.shape))
    with pytest.raises(ValueError, match="destination holds"):
        kv.evict(cache, lens, mass, to, torch.zeros((2, 2, 65), device="cuda"), 65, recent=2)
    unaligned = torch.zeros(cache.k.numel() + 2, device="cuda")[2:].view(cache.k.shape)
    with pytest.raises(ValueError, match="16-byte"):
        kv.attend(kv.PagedKV(unaligned, unaligned, cache.table), q, lens)


def test_empty_calls(cuda):
    cache, q = _case(1, [64, 64], 2, 2, 64, 16, F32, F32)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert kv.attend(cache, q[:0], none).shape == (0, 4, 64)
    assert kv.append(cache, torch.zeros((0, 512), device="cuda"), none, 4, 1e4).shape == (0, 4, 64)
    pages, counts = kv.select_pages(cache, kv.PageBounds.new(cache), q[:0], none, 4)
    assert pages.shape == (0, 2, 4) and counts.shape == (0, 2)
    out = kv.attend(cache, q, _i32([0, 0]))
    assert torch.all(out == 0)


def test_streams_and_graph_replay(cuda):
    """Captured once, replayed with other lengths, tables and queries; two graphs that share nothing; another stream."""
    lens = [300, 45]
    cache, q = _case(12, lens, 2, 4, 128, 16, BF16, BF16)
    ns = _i32(lens)
    kv.attend(cache, q, ns)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(kv.attend(cache, q, ns))
        graphs.append(g)
    for new in ([300, 45], [17, 0], [1, 33]):
        ns.copy_(_i32(new))
        q.copy_(torch.randn(q.shape).to(BF16))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for out in outs:
            _check_attend(cache, q, new, out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = kv.attend(cache, q, ns)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, outs[0])


def test_append_into_other_places(cuda):
    """slots apart from positions: the angle goes by one, the place by the other."""
    k = torch.zeros((4, 1, 16, 64), device="cuda")
    cache = kv.PagedKV(k, k.clone(), _i32([[2, 0]]))
    x = torch.randn((2, 3 * 64), device="cuda")
    kv.append(cache, x, _i32([900, 901]), 1, 1e4, seqs=_i32([0, 0]), slots=_i32([3, 17]))
    other = kv.PagedKV(torch.zeros((64, 1, 16, 64), device="cuda"), torch.zeros((64, 1, 16, 64), device="cuda"),
                       torch.arange(64, dtype=torch.int32, device="cuda")[None])
    kv.append(other, x, _i32([900, 901]), 1, 1e4, seqs=_i32([0, 0]))
    assert torch.equal(k[2, 0, 3], other.k[900 // 16, 0, 900 % 16]) and torch.equal(k[0, 0, 1], other.k[901 // 16, 0, 901 % 16])
    assert int((k != 0).any(-1).sum()) == 2


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_run_of_them_together(cuda, dtype):
    """Prompts appended and attended with their weights, sequences cut by
    them, then new tokens: against attention over the kept keys in 64 bits."""
    gen = torch.Generator().manual_seed(11)
    S, KH, H, d, ps, theta = 3, 2, 6, 64, 16, 1e4
    lens, budget, sinks, recent = [200, 90, 37], 64, 4, 16
    pages = 60
    k, v = (torch.full((pages, KH, ps, d), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    ids = torch.randperm(pages, generator=gen).to(torch.int32)
    table, to_table = ids[:3 * 14].view(3, 14).cuda(), ids[42:54].view(3, 4).cuda()
    cache, to = kv.PagedKV(k, v, table), kv.PagedKV(k, v, to_table)
    seqs = [s for s, n in enumerate(lens) for _ in range(n)]
    pos = [p for n in lens for p in range(n)]
    qkv = torch.randn((len(seqs), (H + 2 * KH) * d), generator=gen).to(dtype).cuda()
    q = kv.append(cache, qkv, _i32(pos), H, theta, seqs=_i32(seqs))
    rows = torch.zeros((len(seqs), KH, 224), device="cuda")
    seen = [p + 1 for p in pos]
    out = kv.attend(cache, q, _i32(seen), seqs=_i32(seqs), mass=rows)
    pick = [0, 7, 199, 200, 289, 290, 326]
    _check_attend(cache, q[pick], [seen[i] for i in pick], out[pick], seqs=[seqs[i] for i in pick])
    mass = torch.stack([rows[[i for i, s in enumerate(seqs) if s == r]].sum(0) for r in range(S)])
    to_mass = torch.zeros((S, KH, 64), device="cuda")
    kept, new = kv.evict(cache, _i32(lens), mass, to, to_mass, budget, sinks=sinks, recent=recent)
    assert new.tolist() == [64, 64, 37]
    host = mass.cpu().numpy()
    old = {s: (tokens(k, table, s, lens[s]), tokens(v, table, s, lens[s])) for s in range(S)}
    for s in range(S):
        for h in range(KH):
            assert kept[s, h, :new[s]].tolist() == choose(host[s, h], lens[s], budget, sinks, recent)
    # 60 places more of every table: new tokens go behind the kept ones, at their own positions
    table2 = torch.cat([to_table, ids[54:60].view(3, 2).cuda()], 1)
    cache2 = kv.PagedKV(k, v, table2)
    step = torch.randn((S, (H + 2 * KH) * d), generator=gen).to(dtype).cuda()
    q2 = kv.append(cache2, step, _i32(lens), H, theta, slots=new)
    mass2 = torch.zeros((S, KH, 96), device="cuda")
    mass2[:, :, :64] = to_mass
    mass0 = mass2.clone()
    out2 = kv.attend(cache2, q2, new + 1, mass=mass2)
    _check_attend(cache2, q2, (new + 1).tolist(), out2, mass=mass2, mass0=mass0)
    for s in range(S):
        got_k, got_v = tokens(k, table2, s, int(new[s])), tokens(v, table2, s, int(new[s]))
        for h in range(KH):
            at = kept[s, h, :new[s]].cpu().numpy()
            assert np.array_equal(got_k[h], old[s][0][h][at]) and np.array_equal(got_v[h], old[s][1][h][at])
    # and sparsely, with room for every page: the same keys
    bounds = kv.PageBounds.new(cache2)
    kv.page_bounds(cache2, bounds, new + 1, _i32([0, 0, 0]))
    sel, counts = kv.select_pages(cache2, bounds, q2, new + 1, 6)
    _check_attend(cache2, q2, (new + 1).tolist(), kv.attend(cache2, q2, new + 1, pages=sel, counts=counts))
    cache.check(), cache2.check()


@pytest.mark.parametrize(("cache_dtype", "q_dtype"), [(F32, F32), (BF16, F32), (BF16, BF16), (F32, BF16)])
@pytest.mark.parametrize(("heads", "kv_heads", "d", "ps"), [(4, 2, 64, 16), (40, 8, 96, 24), (3, 1, 24, 8)])
def test_append_of_a_prompt_is_that_of_its_parts(cuda, cache_dtype, q_dtype, heads, kv_heads, d, ps):
    """Long calls take several tokens a block, and heads in rounds: bit for bit what short calls leave."""
    gen = torch.Generator().manual_seed(heads)
    n, width = 1187, -(-1200 // ps)  # no multiple of the tokens a block takes
    shape = (width + 1, kv_heads, ps, d)
    table = torch.randperm(width + 1, generator=gen)[:width].to(torch.int32)[None].cuda()
    qkv = torch.randn((n, (heads + 2 * kv_heads) * d), generator=gen).to(q_dtype).cuda()
    pos = torch.randperm(1200, generator=gen)[:n].to(torch.int32).cuda()
    pos[7], pos[n - 1] = width * ps, -1  # outside the table: left out, the tokens beside them written
    got = []
    for cuts in ([0, n], [0, 400, 800, n]):
        k, v = (torch.full(shape, 9.0, dtype=cache_dtype, device="cuda") for _ in range(2))
        cache = kv.PagedKV(k, v, table)
        q = [kv.append(cache, qkv[a:b], pos[a:b], heads, 1e4, seqs=_i32([0] * (b - a))) for a, b in zip(cuts, cuts[1:])]
        got.append((torch.cat(q), k, v))
        with pytest.raises(ValueError, match="a length, position"):
            cache.check()
    for one, parts in zip(*got):
        assert torch.equal(one, parts)
    assert int((got[0][2] != 9).any(-1).sum()) == (n - 2) * kv_heads


@pytest.mark.parametrize(("cache_dtype", "q_dtype"), [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize(("d", "ps"), [(32, 24), (64, 16), (128, 7), (192, 64), (256, 8)])
def test_attend_wide_groups_over_many_tiles(cuda, cache_dtype, q_dtype, d, ps):
    """Two tiles of queries, units that end within a block's run and units that several blocks share."""
    lens = [3000, 1, 700, 0, 2049]
    cache, q = _case(d, lens, 2, 11, d, ps, cache_dtype, q_dtype)
    out = kv.attend(cache, q, _i32(lens))
    _check_attend(cache, q, lens, out)
    wide = torch.full((5, 40000), -1, dtype=torch.int32, device="cuda")  # a longest row that rules clusters out
    wide[:, :cache.width] = cache.table
    _check_attend(cache, q, lens, kv.attend(kv.PagedKV(cache.k, cache.v, wide), q, _i32(lens)))
    cache.check()


def test_calls_of_one_cache_on_two_streams(cuda):
    """Nothing is shared by two calls under way at once, captured or not."""
    lens = [5000, 333, 40, 2100]
    cache, q = _case(8, lens, 2, 4, 128, 16, BF16, BF16)
    ns, bounds = _i32(lens), kv.PageBounds.new(cache)
    kv.page_bounds(cache, bounds, ns, _i32([0] * 4))
    want = kv.attend(cache, q, ns)
    want_pages, _ = kv.select_pages(cache, bounds, q, ns, 9)
    streams, outs, graphs = [torch.cuda.Stream() for _ in range(2)], [], []
    torch.cuda.synchronize()
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append((kv.attend(cache, q, ns), kv.select_pages(cache, bounds, q, ns, 9)[0]))
    torch.cuda.synchronize()
    for _ in streams:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(5):
                outs.append((kv.attend(cache, q, ns), kv.select_pages(cache, bounds, q, ns, 9)[0]))
        graphs.append(g)
    for s, g in zip(streams, graphs):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    for out, pages in outs:
        assert torch.equal(out, want) and torch.equal(pages, want_pages)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("wide", [False, True])
def test_mass_of_spoilt_rows(cuda, dtype, wide):
    """A bad page spoils a row's mass up to its length, a bad length or sequence, or one beyond the mass, all of it;
    the rows beside them grow as ever. By a cluster a unit and (a table too wide for that) by equal shares."""
    cache, q = _case(13, [100] * 7, 1, 3, 64, 16, dtype, dtype)
    table = torch.full((7, 40000 if wide else cache.width), -1, dtype=torch.int32, device="cuda")
    table[:, :cache.width] = cache.table
    table[1, 6] = cache.num_pages
    cache = kv.PagedKV(cache.k, cache.v, table)
    given = [100, 100, -1, 113 if not wide else 640001, 100, 90, 0]
    mass = torch.rand((7, 1, 112), device="cuda")
    mass0 = mass.clone()
    out = kv.attend(cache, q, _i32(given), seqs=_i32([0, 1, 2, 3, 7, 5, 6]), mass=mass)
    for r in (1, 2, 3, 4):
        assert torch.isnan(out[r]).all() and torch.isnan(mass[r, 0, :100]).all(), r
    assert torch.equal(mass[1, :, 100:], mass0[1, :, 100:])
    for r in (2, 3, 4):
        assert torch.isnan(mass[r]).all(), r
    for r in (0, 5, 6):
        _check_attend(cache, q[r:r + 1], [given[r]], out[r:r + 1], seqs=[r], mass=mass[r:r + 1], mass0=mass0[r:r + 1])
    with pytest.raises(ValueError, match="page id outside the pool, a length.*, a sequence"):
        cache.check()
    short = mass0[:, :, :99].clone()  # a row longer than the mass has room for
    out = kv.attend(cache, q, _i32([100, 10, 0, 99, 5, 90, 0]), mass=short)
    assert torch.isnan(out[0]).all() and torch.isnan(short[0]).all()
    assert not torch.isnan(out[1:]).any() and not torch.isnan(short[1:]).any()
    with pytest.raises(ValueError, match="a length"):
        cache.check()


def test_pools_of_shared_memory_are_not_written(cuda):
    """k and v in one place are read as they are, and refused where a call would write both there."""
    cache, q = _case(14, [40, 9], 2, 2, 64, 16, F32, F32)
    lens = _i32([40, 9])
    table = cache.table.clone()
    one = kv.PagedKV(cache.k, cache.k, table)
    _check_attend(one, q, [40, 9], kv.attend(one, q, lens))
    shifted = kv.PagedKV(cache.k[:-1], cache.k[1:], table)
    to_mass = torch.zeros((2, 2, 8), device="cuda")
    for pools in (one, shifted):
        with pytest.raises(ValueError, match="k and v share memory"):
            kv.append(pools, torch.zeros((2, 8 * 64), device="cuda"), _i32([0, 0]), 4, 1e4)
        with pytest.raises(ValueError, match="k and v share memory"):
            kv.evict(cache, lens, torch.zeros((2, 2, 64), device="cuda"), pools, to_mass, 8, recent=2)
    pool = torch.zeros((4, 2, 2, 16, 64), device="cuda")  # a page's keys and values side by side
    both = kv.PagedKV(pool[:, 0], pool[:, 1], _i32([[1, 3], [2, 0]]))
    x = torch.randn((2, 8 * 64), device="cuda")
    kv.append(both, x, _i32([17, 2]), 4, 1e4)
    assert torch.equal(pool[3, 1, :, 1], x[0].view(8, 64)[6:]) and torch.equal(pool[2, 1, :, 2], x[1].view(8, 64)[6:])
    assert int((pool != 0).any(-1).sum()) == 8
    both.check()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize(("group", "d", "ps"), [(1, 128, 16), (4, 64, 32), (8, 80, 8)])
def test_select_follows_the_unquantised_bounds(cuda, dtype, group, d, ps):
    """A page that is left out allows no greater product than one that is taken, but for the codes' rounding: half a
    step of a key's code times the query's size, half a step of the query's times the key's, a quarter of both."""
    lens = [2000, 1111, 640]
    gen = torch.Generator().manual_seed(d + group)
    k, v, table = make_cache(gen, lens, 2, d, ps, dtype)
    strong = 1.0 + 4.0 * (torch.rand(d, generator=gen) < 0.05)  # a few strong channels, as trained keys have
    k *= strong.to(dtype).cuda()
    cache = kv.PagedKV(k, v, table)
    q = torch.randn((3, 2 * group, d), generator=gen).to(dtype).cuda()
    bounds = kv.PageBounds.new(cache)
    kv.page_bounds(cache, bounds, _i32(lens), _i32([0] * 3))
    budget = 12
    pages, counts = kv.select_pages(cache, bounds, q, _i32(lens), budget, sinks=1, recent=1)
    for r, n in enumerate(lens):
        total = -(-n // ps)
        keys = tokens(k, table, r, n)
        for h in range(2):
            qs = q[r, h * group:(h + 1) * group].double().cpu().numpy()
            lo = np.stack([keys[h, i * ps:(i + 1) * ps].min(0) for i in range(total)])
            hi = np.stack([keys[h, i * ps:(i + 1) * ps].max(0) for i in range(total)])
            allow = np.maximum(qs[:, None] * lo, qs[:, None] * hi).sum(-1).max(0)  # greatest product a key in them can have
            step = np.maximum(np.abs(lo), np.abs(hi)).max(-1) / 127
            t = np.abs(qs).max(-1) / 127
            size = np.maximum(np.abs(lo), np.abs(hi)).sum(-1)
            off = (0.5 * step * np.abs(qs).sum(-1)[:, None] + 0.5 * t[:, None] * size + 0.25 * d * t[:, None] * step).max(0)
            off = off * (1 + 2.0 ** -20)  # the steps and the score's two products are rounded to 32 bits
            taken = [p for p in pages[r, h].tolist() if 0 < p < total - 1]
            left = [p for p in range(1, total - 1) if p not in taken]
            assert len(taken) == budget - 2 and counts[r, h].item() == budget
            assert min(allow[p] + off[p] for p in taken) >= max(allow[p] - off[p] for p in left)
            assert (allow[taken].mean() - allow[left].mean()) > allow[left].std()  # and they are the better ones
    cache.check()
