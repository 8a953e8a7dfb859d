"""GPU: copies of pages and the compaction of places, all layers in one call, bit for bit."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from expertrelay_b200 import kv

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _pools(layers, pages, heads, ps, d, dtype, layout, seqs=1, width=1):
    stored = {"hnd": (layers, pages, heads, ps, d), "nhd": (layers, pages, ps, heads, d),
              "wide": (layers, pages, heads, ps, d + 8), "gaps": (layers, pages + 1, heads + 1, ps, d)}[layout]
    gen = torch.Generator(device="cuda").manual_seed(pages * ps + d)
    both = torch.randn((2, *stored), generator=gen, device="cuda").to(dtype)
    both[0, 0, 0, 0, 0, :3] = float("nan")
    k, v = both
    if layout == "nhd":
        k, v = k.transpose(2, 3), v.transpose(2, 3)
    k, v = k[:, :pages, :heads, :, :d], v[:, :pages, :heads, :, :d]
    return both, k, v, torch.full((seqs, width), -1, dtype=torch.int32, device="cuda")


def _same(a, b):
    bits = torch.int32 if a.dtype == F32 else torch.int16
    return torch.equal(a.contiguous().view(bits), b.contiguous().view(bits))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout", ["hnd", "nhd", "wide", "gaps"])
@pytest.mark.parametrize(("layers", "heads", "ps", "d", "n"), [
    (1, 1, 1, 8, 1), (3, 2, 7, 80, 5), (24, 16, 16, 128, 9), (2, 3, 200, 256, 40), (5, 4, 64, 128, 3),
])
def test_copy_pages(cuda, dtype, layout, layers, heads, ps, d, n):
    for partial in (False, True):
        both, k, v, table = _pools(layers, 2 * n + 1, heads, ps, d, dtype, layout)
        cache = kv.PagedLayers(k, v, table)
        order = np.random.default_rng(n).permutation(2 * n + 1)
        src, dst = order[:n].copy(), order[n:2 * n]
        used = np.arange(n) * 13 % (ps + 1) if partial else np.full(n, ps)
        if n > 2:
            src[1] = -1  # passed over
        want, (wk, wv) = both.clone(), (k, v)
        wk, wv = (w.as_strided(k.shape, k.stride(), k.storage_offset()) for w in (want[0], want[0]))
        wk = want.as_strided(k.shape, k.stride(), k.storage_offset())
        wv = want.as_strided(v.shape, v.stride(), v.storage_offset())
        for a, b, m in zip(src, dst, used):
            if a >= 0:
                wk[:, b, :, :m] = k[:, a, :, :m]
                wv[:, b, :, :m] = v[:, a, :, :m]
        kv.copy_pages(cache, _i32(src.tolist()), _i32(dst.tolist()), used=_i32(used.tolist()) if partial else None)
        assert _same(both, want)
        cache.check()


def test_copy_pages_one_layer_and_many_pairs(cuda):
    both, k, v, table = _pools(2, 2 * 66000, 1, 1, 8, BF16, "hnd")
    cache = kv.PagedKV(k[1], v[1], table)
    want = both.clone()
    want[:, 1, 66000:] = want[:, 1, :66000]
    kv.copy_pages(cache, torch.arange(66000, dtype=torch.int32, device="cuda"),
                  torch.arange(66000, 2 * 66000, dtype=torch.int32, device="cuda"))
    assert _same(both, want)
    kv.copy_pages(cache, _i32([]), _i32([]))
    assert _same(both, want)


def test_bad_pages_are_passed_over(cuda):
    both, k, v, table = _pools(2, 8, 2, 4, 16, F32, "hnd")
    cache, want = kv.PagedLayers(k, v, table), both.clone()
    want[:, :, 5] = want[:, :, 1]
    for src, dst, used, words in (([1, 8], [5, 6], None, "page"), ([1, 2], [5, -1], None, "page"), ([1, 2], [5, 2**31 - 1], None, "page"),
                                  ([1, 2], [5, 6], [4, 5], "length"), ([1, 2], [5, 6], [4, -1], "length")):
        both.copy_(want)
        both[:, :, 5] = 0
        kv.copy_pages(cache, _i32(src), _i32(dst), used=None if used is None else _i32(used))
        assert _same(both, want)
        with pytest.raises(ValueError, match=words):
            cache.check()


def _compacted(k, table, seqs, start, keep, counts, ps):
    want = k.clone()
    for s, a, row, n in zip(seqs, start, keep, counts):
        for j in range(n):
            p, q = a + row[j], a + j
            want[:, table[s][q // ps], :, q % ps] = k[:, table[s][p // ps], :, p % ps]
    return want


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout", ["hnd", "nhd", "wide"])
@pytest.mark.parametrize(("layers", "heads", "ps", "d", "span", "most"), [
    (1, 1, 1, 8, 9, 4), (3, 2, 7, 80, 64, 12), (24, 16, 16, 128, 8, 5), (2, 3, 64, 256, 700, 300), (4, 40, 16, 32, 5, 2),
    (1, 1, 32, 32, 3000, 2100),
])
def test_compact(cuda, dtype, layout, layers, heads, ps, d, span, most):
    rng = np.random.default_rng(span)
    start = [0, 5, 2 * ps, 3 * ps + 1]
    counts = [most, 0, max(1, most // 3), 1]
    keep = [sorted(rng.choice(span, n, replace=False).tolist()) for n in counts]
    keep[2] = list(range(counts[2]))  # nothing moves
    seqs, width = [2, 0, 1, 4], -(-(start[3] + span) // ps)
    both, k, v, table = _pools(layers, 5 * width + 2, heads, ps, d, dtype, layout, 5, width)
    table.copy_(torch.from_numpy(rng.permutation(5 * width).reshape(5, width)))
    cache = kv.PagedLayers(k, v, table)
    lists = torch.full((4, most + 3), -5, dtype=torch.int32, device="cuda")
    for i, row in enumerate(keep):
        lists[i, :len(row)] = _i32(row)
    pages = table.tolist()
    wk, wv = (_compacted(x, pages, seqs, start, keep, counts, ps) for x in (k, v))
    lens = kv.compact(cache, _i32(start), lists[:, :most], _i32(counts), seqs=_i32(seqs))
    assert lens.tolist() == [a + n for a, n in zip(start, counts)]
    assert _same(k, wk) and _same(v, wv)
    cache.check()


@pytest.mark.parametrize("rows", [255, 256, 257, 700])
def test_compact_many_rows(cuda, rows):
    """Lists of all lengths, in every order; a bad one among them."""
    rng = np.random.default_rng(rows)
    ps, width, span = 8, 5, 30
    start = rng.integers(0, 10, rows).tolist()
    counts = rng.integers(0, 13, rows).tolist()
    keep = [sorted(rng.choice(span, n, replace=False).tolist()) for n in counts]
    both, k, v, table = _pools(2, rows * width, 2, ps, 64, BF16, "hnd", rows, width)
    table.copy_(torch.from_numpy(rng.permutation(rows * width).reshape(rows, width)))
    cache = kv.PagedLayers(k, v, table)
    lists = torch.full((rows, 12), -5, dtype=torch.int32, device="cuda")
    for i, row in enumerate(keep):
        lists[i, :len(row)] = _i32(row)
    bad, good = rows // 2, list(counts)
    counts[bad], good[bad] = 13, 0
    pages = table.tolist()
    wk, wv = (_compacted(x, pages, range(rows), start, keep, good, ps) for x in (k, v))
    lens = kv.compact(cache, _i32(start), lists, _i32(counts))
    assert lens.tolist() == [-1 if i == bad else a + n for i, (a, n) in enumerate(zip(start, counts))]
    assert _same(k, wk) and _same(v, wv)
    with pytest.raises(ValueError, match="length"):
        cache.check()


def test_captured_and_on_another_stream(cuda):
    """One graph of a fork and an acceptance, replayed over other pages, lists and counts."""
    ps, width = 4, 6
    both, k, v, table = _pools(3, 3 * width, 2, ps, 32, F32, "hnd", 2, width)
    table.copy_(torch.arange(2 * width).view(2, width))
    cache = kv.PagedLayers(k, v, table)
    src, dst, used = _i32([0, 6]), _i32([12, 13]), _i32([4, 2])
    start, keep, counts = _i32([3, 0]), _i32([[1, 2, 5], [0, 4, 9]]), _i32([3, 2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    was = both.clone()
    with torch.cuda.stream(side):
        kv.copy_pages(cache, src, dst, used=used)
        kv.compact(cache, start, keep, counts)
    torch.cuda.current_stream().wait_stream(side)
    both.copy_(was)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kv.copy_pages(cache, src, dst, used=used)
        lens = kv.compact(cache, start, keep, counts)
    for pairs, lists, n in (([(0, 12, 4), (6, 13, 2)], [[1, 2, 5], [0, 4, 9]], [3, 2]), ([(3, 16, 1), (-1, 0, 4)], [[0, 1, 2], [7, 8, 11]], [1, 3])):
        both.copy_(was)
        for t, new in zip((src, dst, used), zip(*pairs)):
            t.copy_(_i32(list(new)))
        keep.copy_(_i32(lists))
        counts.copy_(_i32(n))
        want = was.clone()
        for a, b, m in pairs:
            if a >= 0:
                want[:, :, b, :, :m] = want[:, :, a, :, :m]
        wk, wv = (_compacted(x, table.tolist(), [0, 1], [3, 0], lists, n, ps) for x in want)
        g.replay()
        assert _same(both[0], wk) and _same(both[1], wv) and lens.tolist() == [3 + n[0], n[1]]
    cache.check()


def test_bad_rows_stay_unwritten(cuda):
    both, k, v, table = _pools(2, 12, 2, 4, 16, F32, "hnd", 3, 4)
    table.copy_(torch.arange(12).reshape(3, 4))
    was = both.clone()
    good = ([3, 4, 2], [[1, 3, 5], [0, 2, 3], [4, 5, 6]], [3, 2, 3])
    for change, words in (({"keep": [1, 3, 3]}, "length"), ({"keep": [1, 3, 2]}, "length"), ({"keep": [-1, 3, 4]}, "length"),
                          ({"keep": [1, 3, 14]}, "length"), ({"keep": [1, 2, 2**31 - 1]}, "length"), ({"count": 4}, "length"),
                          ({"count": -1}, "length"), ({"start": -1}, "length"), ({"start": 2**31 - 1}, "length"),
                          ({"seq": 3}, "sequence"), ({"seq": -1}, "sequence"), ({"page": 12}, "page"), ({"page": -1}, "page")):
        both.copy_(was)
        start, keep, counts = [list(x) for x in good]
        seqs, pages = [0, 1, 2], table.clone()
        if "keep" in change:
            keep[0] = change["keep"]
        if "count" in change:
            counts[0] = change["count"]
        if "start" in change:
            start[0] = change["start"]
        if "seq" in change:
            seqs[0] = change["seq"]
        if "page" in change:
            pages[0, 1] = change["page"]
        cache = kv.PagedLayers(k, v, pages)
        lens = kv.compact(cache, _i32(start), _i32(keep), _i32(counts), seqs=_i32(seqs))
        assert lens.tolist() == [-1, 6, 5], change
        wk = _compacted(was[0], table.tolist(), [1, 2], good[0][1:], good[1][1:], good[2][1:], 4)
        assert _same(both[0], wk), change
        with pytest.raises(ValueError, match=words):
            cache.check()


def test_refusals(cuda):
    both, k, v, table = _pools(2, 6, 2, 4, 16, F32, "hnd", 2, 2)
    cache = kv.PagedLayers(k, v, table)
    i = _i32([0, 1])
    for call, words in (
            (lambda: kv.PagedLayers(k[0], v[0], table), "layers"), (lambda: kv.PagedLayers(k, v[:1], table), "alike"),
            (lambda: kv.PagedLayers(k[:0], v[:0], table), "layers"),
            (lambda: kv.copy_pages(cache, i.long(), i), "src"), (lambda: kv.copy_pages(cache, i, i[:1]), "dst"),
            (lambda: kv.copy_pages(cache, i, i, used=i[:1]), "used"),
            (lambda: kv.copy_pages(kv.PagedLayers(k, k, table), i, i), "share memory"),
            (lambda: kv.copy_pages(kv.PagedLayers(both[0, :1].expand(3, *k.shape[1:]), both[1, :1].expand(3, *k.shape[1:]), table), i, i),
             "share memory"),
            (lambda: kv.compact(cache, i, i, i), "keep"), (lambda: kv.compact(cache, i, i[None].expand(2, 2), i), "keep"),
            (lambda: kv.compact(cache, i[:1], i.view(2, 1), i), "start"), (lambda: kv.compact(cache, i, i.view(2, 1), i[:1]), "counts"),
            (lambda: kv.compact(cache, _i32([0] * 3), _i32([[0]] * 3), _i32([0] * 3)), "seqs"),
            (lambda: kv.compact(kv.PagedLayers(k, k, table), i, i.view(2, 1), i), "share memory")):
        with pytest.raises(ValueError, match=words):
            call()
    assert kv.compact(cache, i[:0], _i32([]).view(0, 3), i[:0]).shape == (0,)
    assert kv.compact(cache, i, _i32([]).view(2, 0), _i32([0, 0])).tolist() == [0, 1]


@pytest.mark.parametrize(("heads", "ps", "d", "dtype", "most"), [
    (4, 32, 128, BF16, 2100), (2, 16, 64, F32, 1300), (1, 64, 8, BF16, 3000), (3, 24, 136, BF16, 500), (1, 16, 248, F32, 260),
    (8, 32, 256, F32, 1100),
])
def test_lists_of_many_batches(cuda, heads, ps, d, dtype, most):
    """Many long lists in many layers at once, so that the warps of a CTA are not abreast: every key and value in its
    place, several times over."""
    rng = np.random.default_rng(most + d)
    layers, rows, span = 6, 24, most + most // 3
    start = rng.integers(0, 3 * ps, rows)
    counts = [most, 0, 1, *rng.integers(most // 2, most + 1, rows - 3).tolist()]
    width = -(-(int(start.max()) + span) // ps)
    both, k, v, table = _pools(layers, rows * width, heads, ps, d, dtype, "hnd", rows, width)
    table.copy_(torch.from_numpy(rng.permutation(rows * width).reshape(rows, width)))
    lists = np.full((rows, most), -1)
    for i, n in enumerate(counts):
        lists[i, :n] = np.sort(rng.choice(span, n, replace=False))
    row, j = (torch.from_numpy(x).cuda() for x in np.nonzero(lists >= 0))
    frm = torch.from_numpy(start[row.cpu()] + lists[lists >= 0]).cuda()
    to = torch.from_numpy(start).cuda()[row] + j
    pages = table.long()
    want = both.clone()
    want[:, :, pages[row, to // ps], :, to % ps] = both[:, :, pages[row, frm // ps], :, frm % ps]
    cache, was = kv.PagedLayers(k, v, table), both.clone()
    args = _i32(start.tolist()), _i32(lists.tolist()), _i32(counts)
    for _ in range(6):
        both.copy_(was)
        lens = kv.compact(cache, *args)
        assert _same(both, want)
        assert lens.tolist() == [int(a) + n for a, n in zip(start, counts)]
    cache.check()


def test_bad_rows_leave_values_too(cuda):
    """Keys and values of a bad row stay as they were, and the other rows' are moved."""
    both, k, v, table = _pools(3, 12, 2, 4, 16, BF16, "hnd", 3, 4)
    table.copy_(torch.arange(12).reshape(3, 4))
    was, start, counts = both.clone(), [3, 4, 2], [3, 2, 3]
    for keep0, page in (([1, 3, 3], None), ([1, 3, 14], None), ([-1, 3, 4], None), ([1, 3, 5], 12), ([1, 3, 5], -1)):
        both.copy_(was)
        keep, pages = [keep0, [0, 2, 3], [4, 5, 6]], table.clone()
        if page is not None:
            pages[0, 1] = page
        cache = kv.PagedLayers(k, v, pages)
        assert kv.compact(cache, _i32(start), _i32(keep), _i32(counts)).tolist() == [-1, 6, 5]
        for pool, old in zip(both, was):
            assert _same(pool, _compacted(old, table.tolist(), [1, 2], start[1:], keep[1:], counts[1:], 4))
        with pytest.raises(ValueError, match="page" if page is not None else "length"):
            cache.check()
