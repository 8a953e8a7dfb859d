"""The paged cache's C entry points without a GPU: every refusal comes before the device is touched."""

from __future__ import annotations

import ctypes as C
from types import SimpleNamespace

import pytest
import torch

from expertrelay_b200 import _lib, kv
from expertrelay_b200.kv_cache import PagedKVCache, PageTable

P = 0x1000  # an address that is never followed


def _cache(**kw):
    base = dict(k=P, v=P, dtype=_lib.DTYPE_BF16, num_pages=8, page_size=16, kv_heads=2, head_dim=64,
                page_stride=2 * 16 * 64, head_stride=16 * 64, slot_stride=64, table=P, seqs=3, table_width=4,
                table_stride=4)
    return _lib.KvCache(**{**base, **kw})


def _io(**kw):
    base = dict(q=P, q_dtype=_lib.DTYPE_BF16, q_stride=4 * 64, out=P, rows=3, heads=4, lens=P, scale=0.1)
    return _lib.KvAttendIO(**{**base, **kw})


def _fails(rc, words):
    assert rc == _lib.ER_EINVAL
    assert words in _lib.last_error(), _lib.last_error()


@pytest.mark.parametrize(("change", "words"), [
    ({"dtype": 2}, "dtype 2"), ({"num_pages": 0}, "0 pages"), ({"page_size": -1}, "-1 positions"),
    ({"kv_heads": 0}, "0 key heads"), ({"head_dim": 60}, "head_dim 60"), ({"head_dim": 264}, "head_dim 264"),
    ({"head_dim": 0}, "head_dim 0"), ({"k": None}, "null"), ({"table": None}, "null"), ({"k": P + 8}, "16-byte"),
    ({"slot_stride": 68}, "16-byte"), ({"seqs": -1}, "-1 x 4"),
])
def test_cache_refusals(change, words):
    L, c = _lib.lib(), _cache(**change)
    _fails(L.er_kv_attend(C.byref(c), C.byref(_io()), None, 0, None), words)
    _fails(L.er_kv_append(C.byref(c), P, 1, 8 * 64, None, P, None, 1, 4, 1e4, P, 1, None, None), words)
    _fails(L.er_kv_page_bounds(C.byref(c), P, P, P, P, None, None), words)
    _fails(L.er_kv_select(C.byref(c), P, 1, 256, 1, 4, None, P, P, P, 4, 0, 0, P, P, None, None), words)
    _fails(L.er_kv_evict(C.byref(c), C.byref(_cache()), P, P, 1, 1, 64, P, 1, 1, 64, 8, 0, 0, P, P, None, None), words)


@pytest.mark.parametrize(("change", "words"), [
    ({"rows": -1}, "rows -1"), ({"heads": 3}, "heads 3 / 2"), ({"heads": 0}, "heads 0"),
    ({"heads": 2**31 - 2, "q_stride": 2**40}, "heads 2147483646"), ({"q_dtype": 7}, "q dtype 7"),
    ({"q_stride": 255}, "row stride 255"), ({"pages": P}, "page lists"), ({"pages": P, "max_pages": 4}, "page lists"),
    ({"pages": P, "counts": P, "max_pages": 4, "mass": P}, "page lists"), ({"mass": P, "mass_len": -1}, "mass_len"),
    ({"rows": 4}, "4 rows, 3 sequences"), ({"out": P + 8}, "16-byte"), ({"q": None}, "null"), ({"out": None}, "null"), ({"lens": None}, "null"),
])
def test_attend_refusals(change, words):
    _fails(_lib.lib().er_kv_attend(C.byref(_cache()), C.byref(_io(**change)), None, 0, None), words)


def test_append_refusals():
    L, c = _lib.lib(), _cache()
    args = [C.byref(c), P, 1, 8 * 64, None, P, None, 1, 4, 1e4, P, 1, None, None]
    for at, value, words in [(1, None, "null"), (2, 5, "dtypes 5"), (3, 8 * 64 - 1, "row stride"), (5, None, "null"),
                             (7, -1, "n -1"), (8, 0, "heads 0"), (8, 2**31 - 1, "heads"), (9, 0.0, "theta 0"), (9, float("nan"), "theta"),
                             (10, None, "null"), (11, 9, "9")]:
        _fails(L.er_kv_append(*[value if i == at else x for i, x in enumerate(args)]), words)


def test_select_refusals():
    L, c = _lib.lib(), _cache()
    args = [C.byref(c), P, 1, 256, 1, 4, None, P, P, P, 4, 1, 1, P, P, None, None]
    for at, value, words in [(1, None, "null"), (2, 3, "q dtype"), (3, 8, "row stride"), (4, -2, "rows -2"),
                             (5, 5, "heads 5"), (7, None, "null"), (8, P + 8, "16-byte"), (10, 0, "budget 0"),
                             (11, 4, "budget 4"), (12, -1, "budget 4"), (4, 4, "4 rows, 3 sequences")]:
        _fails(L.er_kv_select(*[value if i == at else x for i, x in enumerate(args)]), words)
    args[0] = C.byref(_cache(table_width=600000))
    _fails(L.er_kv_select(*args), "table of 600000 pages")
    args[0], args[3], args[5] = C.byref(c), 130 * 64, 130
    _fails(L.er_kv_select(*args), "65 queries a key head")


def test_evict_refusals():
    L = _lib.lib()
    def call(frm=None, to=None, **kw):
        a = dict(lens=P, mass=P, mass_len=64, to_mass=P, to_mass_len=64, budget=8, sinks=1, recent=1, kept=P, out=P + 64)
        a.update(kw)
        return L.er_kv_evict(C.byref(frm or _cache()), C.byref(to or _cache()), a["lens"], a["mass"], 1, 1,
                             a["mass_len"], a["to_mass"], 1, 1, a["to_mass_len"], a["budget"], a["sinks"], a["recent"],
                             a["kept"], a["out"], None, None)
    for other in ({"dtype": 0, "slot_stride": 64}, {"kv_heads": 1}, {"head_dim": 32}, {"seqs": 2}):
        _fails(call(to=_cache(**other)), "differ")
    _fails(call(budget=0), "budget 0")
    _fails(call(sinks=8), "budget 8")
    _fails(call(budget=65), "destination holds 64")
    _fails(call(to_mass_len=7), "7 weights")
    _fails(call(out=P), "lens_out is lens")
    _fails(call(mass_len=500000), "500000 weights")
    for name in ("lens", "mass", "to_mass", "kept", "out"):
        _fails(call(**{name: None}), "null")


def test_limits_of_sequences_and_key_heads():
    L, c = _lib.lib(), _cache(seqs=65536)
    _fails(L.er_kv_page_bounds(C.byref(c), P, P, P, P, None, None), "65536 sequences")
    _fails(L.er_kv_evict(C.byref(c), C.byref(c), P, P, 1, 1, 64, P, 1, 1, 64, 8, 0, 0, P, P + 64, None, None), "65536 sequences")
    c = _cache(kv_heads=1025)
    _fails(L.er_kv_attend(C.byref(c), C.byref(_io(heads=1025, q_stride=2**30)), None, 0, None), "1025 key heads")
    _fails(L.er_kv_page_bounds(C.byref(c), P, P, P, P, None, None), "1025 key heads")


def test_nothing_to_do_is_fine():
    L = _lib.lib()
    assert L.er_kv_attend(C.byref(_cache()), C.byref(_io(rows=0)), None, 0, None) == _lib.ER_OK
    assert L.er_kv_append(C.byref(_cache()), P, 1, 512, None, P, None, 0, 4, 1e4, P, 1, None, None) == _lib.ER_OK
    assert L.er_kv_page_bounds(C.byref(_cache(seqs=0)), P, P, P, P, None, None) == _lib.ER_OK


def test_weights_that_share_memory():
    a = torch.zeros(4 * 2 * 3 * 10)
    share = kv._share
    two = a.view(4, 2, 3, 10)
    assert not share(two[0], two[1]) and not share(two[3], two[0])       # one behind the other
    assert not share(two.transpose(0, 1)[0][:, :, :4], two.transpose(0, 1)[1])  # layers of one array
    assert share(two[0], two[0]) and share(two[0], two[0][:, :, :4]) and share(two[0][:, :, 1:], two[0])
    assert share(a[:60].view(2, 3, 10), a[5:65].view(2, 3, 10)) and share(a[:60].view(2, 3, 10), a[40:58].view(2, 3, 3))
    assert not share(two[0], torch.zeros(2, 3, 10)) and not share(two[:, :0, 0], two[:, :, 0])


def test_page_table_gives_and_takes_pages():
    t = PageTable(3, 4, 7, 16)
    pos, slots = t.extend([0] * 17 + [2])
    assert pos.tolist() == slots.tolist() == [*range(17), 0]
    assert t.length.tolist() == t.position.tolist() == [17, 0, 1] and len(t.free) == 4
    pages = [p for p in t.table.ravel() if p >= 0]
    assert len(pages) == len(set(pages)) == 3
    pos, slots = t.extend([2, 0, 2])  # interleaved
    assert pos.tolist() == [1, 17, 2] and slots.tolist() == [1, 17, 2]
    # evicted to 5 places: positions go on, places start over
    t.replace(0, t.take(1), 5)
    pos, slots = t.extend([0])
    assert pos.tolist() == [18] and slots.tolist() == [5]
    t.release(0)
    assert t.length.tolist() == [0, 0, 3] and t.position.tolist() == [0, 0, 3] and len(t.free) == 6
    assert sorted(t.free + [int(p) for p in t.table.ravel() if p >= 0]) == list(range(7))


def test_page_table_refusals_change_nothing():
    t = PageTable(2, 4, 5, 16)
    t.extend([0] * 48)
    before = (t.table.copy(), t.length.copy(), t.position.copy(), list(t.free))
    for seqs, words in [([0] * 17, "sequence length 65 exceeds"), ([1] * 33, "out of pages"), ([2], "outside"), ([-1], "outside")]:
        with pytest.raises(ValueError, match=words):
            t.extend(seqs)
    with pytest.raises(ValueError, match="out of pages"):
        t.take(3)
    assert (t.table == before[0]).all() and (t.length == before[1]).all() and (t.position == before[2]).all()
    assert t.free == before[3]
    assert [len(x) for x in t.extend([])] == [0, 0]
    with pytest.raises(ValueError, match="at least one"):
        PageTable(1, 0, 1, 16)


def test_page_table_takes_an_extension_back():
    t = PageTable(4, 8, 20, 4)
    t.extend([0] * 5 + [2] * 4)
    t.release(0)
    t.extend([3] * 3 + [2])
    t.replace(2, t.take(1), 3)  # evicted: positions and places differ
    before = (t.table.copy(), t.length.copy(), t.position.copy(), list(t.free))
    for seqs in ([2], [2, 3, 2, 0, 3, 3, 3, 0], [1] * 9, [], [0] * 32, [3, 2, 1, 0]):
        t.extend(seqs)
        t.shrink(seqs)
        assert (t.table == before[0]).all() and (t.length == before[1]).all() and (t.position == before[2]).all()
        assert t.free == before[3]  # in order, so that a retry gets the same pages


def test_a_sequence_keeps_some_of_its_own_pages():
    t = PageTable(2, 4, 8, 16)
    t.extend([0] * 64 + [1] * 64)
    own = [int(p) for p in t.table[0, :2]]
    rest = [int(p) for p in t.table[0, 2:]]
    t.replace(0, own, 20)
    assert t.table[0].tolist() == [*own, -1, -1] and sorted(t.free) == sorted(rest)
    assert t.length.tolist() == [20, 64] and t.position.tolist() == [64, 64]


def test_pools_that_share_memory():
    def share(k, v):
        assert k.stride() == v.stride() and kv._apart(k.shape, k.stride())
        got = kv._meet((v.data_ptr() - k.data_ptr()) // k.element_size(), k.shape, k.stride())
        at = torch.arange(a.numel()).view(a.shape)  # and as counted place by place
        both = [set(torch.as_strided(at, x.shape, x.stride(), x.storage_offset()).flatten().tolist()) for x in (k, v)]
        assert got == bool(both[0] & both[1])
        return got

    a = torch.zeros(6 * 2 * 3 * 4 * 8)
    both = a.view(6, 2, 3, 4, 8)  # keys and values of a page side by side
    assert not share(both[:, 0], both[:, 1]) and not share(both[:, 1], both[:, 0])
    wide = a.view(6, 3, 4, 16)  # or of a slot
    assert not share(wide[..., :8], wide[..., 8:])
    assert not share(both[:3, 0], both[3:, 0])
    k = a.view(12, 3, 4, 8)
    assert share(k, k) and share(k[:8], k[4:]) and share(wide[..., :8], wide[..., 4:12])
    assert not share(k[0:6:2], k[3:9:2]) and share(k[0:6:2], k[4:10:2])  # every other page, from an odd or an even one on
    assert not share(k[0:9:3], k[1:10:3]) and share(k[3:12:3], k[0:9:3]) and not share(k[:, 2:], k[:, 1:2])
    assert not share(k[..., 2:3, :], k[..., 0:1, :]) and share(k[..., 1:3, :], k[..., 0:2, :])


def test_a_sequence_outside_the_table_is_not_another_one():
    t = PageTable(3, 4, 7, 16)
    t.extend([2] * 20)
    for seq in (-1, 3):
        with pytest.raises(ValueError, match="outside"):
            t.release(seq)
    assert t.length.tolist() == [0, 0, 20] and len(t.free) == 5
    with pytest.raises(ValueError, match="one for each row"):
        t.extend([[0, 1]])


@pytest.mark.parametrize("change", [{"page_size": 0}, {"page_size": -4}, {"max_seq": 0}, {"seqs": 0}, {"pages": 0}])
def test_a_cache_of_nothing_is_refused(change):
    shape = SimpleNamespace(num_layers=1, num_kv_heads=1, head_dim=8)
    args = {"seqs": 1, "max_seq": 8, "page_size": 4, "device": "cpu", **change}
    with pytest.raises(ValueError, match="at least one"):
        PagedKVCache(shape, **args)
