"""Several continuations of a text, without a GPU: pages that sequences share, drafts, and the refusals of the C
entry points behind them, which come before the device is touched."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from expertrelay_b200 import _lib, draft
from expertrelay_b200.kv_cache import PageTable

P = 0x1000  # an address that is never followed


def _cache(**kw):
    base = dict(k=P, v=P, dtype=_lib.DTYPE_BF16, num_pages=8, page_size=16, kv_heads=2, head_dim=64,
                page_stride=2 * 16 * 64, head_stride=16 * 64, slot_stride=64, table=P, seqs=3, table_width=4,
                table_stride=4)
    return _lib.KvCache(**{**base, **kw})


def _fails(rc, words):
    assert rc == _lib.ER_EINVAL
    assert words in _lib.last_error(), _lib.last_error()


def _tree(**kw):
    base = dict(q=P, q_dtype=_lib.DTYPE_BF16, q_stride=4 * 64, out=P, rows=5, heads=4, trees=2, starts=P, parents=P,
                lens=P, scale=0.1)
    return _lib.KvTreeIO(**{**base, **kw})


CACHES = [({"dtype": 2}, "dtype 2"), ({"num_pages": 0}, "0 pages"), ({"page_size": -1}, "-1 positions"),
          ({"kv_heads": 0}, "0 key heads"), ({"kv_heads": 1025}, "1025 key heads"), ({"head_dim": 60}, "head_dim 60"),
          ({"head_dim": 264}, "head_dim 264"), ({"k": None}, "null"), ({"table": None}, "null"), ({"k": P + 8}, "16-byte"),
          ({"slot_stride": 68}, "16-byte"), ({"seqs": -1}, "-1 x 4")]


@pytest.mark.parametrize(("change", "words"), CACHES)
def test_cache_refusals(change, words):
    L, c = _lib.lib(), _cache(**change)
    _fails(L.er_kv_tree(C.byref(c), C.byref(_tree(heads=4 if c.kv_heads < 1000 else 1025, q_stride=2**30)), None, 0, None), words)
    assert L.er_kv_tree_workspace_bytes(C.byref(c), C.byref(_tree(heads=4 if c.kv_heads < 1000 else 1025, q_stride=2**30))) == 0
    _fails(L.er_kv_copy_pages(C.byref(c), 1, 0, P, P, None, 1, None, None), words)
    _fails(L.er_kv_compact(C.byref(c), 1, 0, None, P, P, 4, 4, P, 1, None, None, None), words)


@pytest.mark.parametrize(("change", "words"), [
    ({"rows": -1}, "-1 rows"), ({"trees": -1}, "-1 trees"), ({"heads": 3}, "heads 3 / 2"), ({"heads": 0}, "heads 0"),
    ({"heads": 2**31 - 2, "q_stride": 2**40}, "heads 2147483646"), ({"trees": 4097, "seqs": P}, "4097 trees"),
    ({"q_dtype": 7}, "q dtype 7"), ({"q_stride": 255}, "row stride 255"), ({"trees": 4}, "4 trees, 3 sequences"),
    ({"out": P + 8}, "16-byte"), ({"q": None}, "null"), ({"out": None}, "null"), ({"lens": None}, "null"),
    ({"starts": None}, "null"), ({"parents": None}, "null"),
])
def test_tree_refusals(change, words):
    _fails(_lib.lib().er_kv_tree(C.byref(_cache()), C.byref(_tree(**change)), None, 0, None), words)


def test_a_tree_call_without_its_arguments():
    L = _lib.lib()
    _fails(L.er_kv_tree(C.byref(_cache()), None, None, 0, None), "null io")
    _fails(L.er_kv_tree(None, C.byref(_tree()), None, 0, None), "null")
    for nothing in ({"rows": 0}, {"trees": 0}):
        assert L.er_kv_tree(C.byref(_cache()), C.byref(_tree(**nothing)), None, 0, None) == _lib.ER_OK
        assert L.er_kv_tree_workspace_bytes(C.byref(_cache()), C.byref(_tree(**nothing))) == 0


def test_copy_refusals():
    L, c = _lib.lib(), _cache()
    args = [C.byref(c), 2, 1 << 16, P, P, None, 3, None, None]
    for at, value, words in [(1, 0, "0 layers"), (1, 32768, "32768 layers"), (2, 12, "16-byte"), (3, None, "null"), (4, None, "null"),
                             (6, -1, "n -1")]:
        _fails(L.er_kv_copy_pages(*[value if i == at else x for i, x in enumerate(args)]), words)
    args[6] = 0
    assert L.er_kv_copy_pages(*args) == _lib.ER_OK
    args[0] = C.byref(_cache(page_size=2**30))
    _fails(L.er_kv_copy_pages(*args), "above 16 GB")


def test_compact_refusals():
    L, c = _lib.lib(), _cache()
    args = [C.byref(c), 2, 1 << 16, None, P, P, 4, 4, P, 3, P, None, None]
    for at, value, words in [(1, -1, "-1 layers"), (2, 4, "16-byte"), (4, None, "null"), (5, None, "null"), (6, 3, "stride 3"),
                             (7, -1, "-1 entries"), (8, None, "null"), (9, -2, "-2 rows"), (9, 4, "4 rows, 3 sequences")]:
        _fails(L.er_kv_compact(*[value if i == at else x for i, x in enumerate(args)]), words)
    args[9] = 0
    assert L.er_kv_compact(*args) == _lib.ER_OK


def test_beam_refusals():
    L = _lib.lib()
    args = [P, _lib.DTYPE_F32, 100, P, 2, 3, 100, 4, P, P, P, None, 0, None]
    for at, value, words in [(0, None, "null"), (1, 9, "dtype 9"), (2, 99, "row stride 99"), (3, None, "null"), (4, -1, "-1 batches"),
                             (5, 0, "0 beams"), (5, 1025, "1025 beams"), (6, 0, "vocabulary of 0"), (7, 0, "count 0"), (7, 129, "count 129"),
                             (4, 21846, "65538 rows"), (8, None, "null"), (9, None, "null"), (10, None, "null")]:
        _fails(L.er_beam_select(*[value if i == at else x for i, x in enumerate(args)]), words)
    args[5], args[6], args[2] = 1, 3, 3
    _fails(L.er_beam_select(*args), "count 4")
    args[4], args[7] = 0, 3
    assert L.er_beam_select(*args) == _lib.ER_OK
    for sizes in ((0, 3, 100, 4), (2, 0, 100, 4), (2, 3, 100, 500)):
        assert L.er_beam_workspace_bytes(*sizes) == 0


@pytest.mark.parametrize("seed", range(6))
def test_sequences_share_pages_and_keep_their_places(seed):
    rng = np.random.default_rng(seed)
    seqs, ps, pages = 5, int(rng.integers(1, 6)), 30
    t, texts, store, n = PageTable(seqs, 12, pages, ps), [[] for _ in range(seqs)], {}, 0

    def whole():
        named = np.bincount(t.table[t.table >= 0], minlength=pages)
        assert (named == t.uses).all() and sorted(t.free) == np.flatnonzero(named == 0).tolist()
        for s, text in enumerate(texts):
            assert t.length[s] == t.position[s] == len(text)
            assert [store[int(t.table[s, i // ps]), i % ps] for i in range(len(text))] == text
            assert (t.table[s, -(-len(text) // ps):] == -1).all()

    for _ in range(120):
        do = rng.integers(0, 4)
        before = (t.table.copy(), t.length.copy(), t.position.copy(), list(t.free), t.uses.copy())
        try:
            if do <= 1:
                rows = rng.integers(0, seqs, rng.integers(1, 9))
                _, slots = t.extend(rows)
                for s, slot in zip(rows.tolist(), slots.tolist()):
                    assert slot == len(texts[s])
                    store[int(t.table[s, slot // ps]), slot % ps] = n
                    texts[s].append(n)
                    n += 1
                if do == 1:  # the last places of one of them go
                    s = int(rows[0])
                    cut = int(rng.integers(0, np.count_nonzero(rows == s) + 1))
                    t.shrink([s] * cut)
                    texts[s] = texts[s][:len(texts[s]) - cut]
            elif do == 2:
                some = rng.permutation(seqs)[:rng.integers(0, seqs + 1)]
                parents = rng.integers(0, seqs, len(some))
                src, dst, used = t.reorder(some, parents)
                assert not set(src) & set(dst) and len(set(dst)) == len(dst)
                for a, b, u in zip(src, dst, used):
                    for i in range(u):
                        store[b, i] = store[a, i]
                texts = [list(texts[parents[some.tolist().index(s)]]) if s in some else texts[s] for s in range(seqs)]
            else:
                s = int(rng.integers(0, seqs))
                t.release(s)
                texts[s] = []
        except ValueError as error:
            assert "out of pages" in str(error) or "exceeds" in str(error)
            assert all(np.array_equal(a, b) for a, b in zip(before, (t.table, t.length, t.position, t.free, t.uses)))
        whole()


def test_one_child_keeps_the_last_page():
    t = PageTable(4, 4, 8, 4)
    t.extend([0] * 6)
    assert t.reorder([1], [0]) == ([int(t.table[0, 1])], [int(t.table[1, 1])], [2])  # its parent stays
    assert t.table[0, 0] == t.table[1, 0] and t.uses[t.table[0, 0]] == 2
    page = int(t.table[1, 1])
    assert t.reorder([0, 1], [1, 1])[0] == [page] and page in t.table[:2, 1]  # one of the two has it on
    assert t.reorder([2, 0, 1], [0, 3, 3]) == ([], [], [])  # handed on whole
    assert t.length.tolist() == [0, 0, 6, 0] and len(t.free) == 6
    t.extend([2] * 2)
    assert t.reorder([0, 1, 3], [2, 2, 2]) == ([], [], []) and len(t.free) == 6  # full pages only: nothing to copy


def test_a_text_that_repeats_itself():
    assert draft.from_text([1, 2, 3]) == ([], []) and draft.from_text([]) == ([], []) and draft.from_text([4]) == ([], [])
    assert draft.from_text([1, 2, 3, 9, 1, 2, 3], length=2) == ([9, 1], [-1, 0])
    tokens, parents = draft.from_text([1, 2, 5, 1, 2, 6, 7, 1, 2, 5, 8, 1, 2], length=3)
    assert tokens == [5, 8, 1, 6, 7, 1, 1, 2] and parents == [-1, 0, 1, -1, 3, 4, 0, 6]
    assert draft.from_text([7, 7, 7], length=8) == ([7], [-1])
    long = list(range(50)) * 3
    tokens, parents = draft.from_text(long, nodes=5, length=20)
    assert tokens == [0, 1, 2, 3, 4] and parents == [-1, 0, 1, 2, 3]
    assert all(p < i for i, p in enumerate(parents))


def _from_text(text, nodes, length, match):
    """draft.from_text by its definition."""
    tokens, parents, children, n = [], [], {}, len(text)
    for m in range(min(match, n - 1), 0, -1):
        for at in range(n - m - 1, -1, -1):
            parent = -1
            for t in text[at + m:at + m + length] if text[at:at + m] == text[n - m:] else ():
                if (parent, t) not in children:
                    if len(tokens) == nodes:
                        return tokens, parents
                    children[parent, t] = len(tokens)
                    tokens.append(t)
                    parents.append(parent)
                parent = children[parent, t]
        if tokens:
            break
    return tokens, parents


class _Counted(list):
    """A list that counts how often its elements are asked for, and those of its copies."""

    asked = [0]

    def __getitem__(self, at):
        self.asked[0] += 1
        got = super().__getitem__(at)
        return _Counted(got) if isinstance(at, slice) else got


def test_drafts_from_short_texts_of_few_tokens():
    rng = np.random.default_rng(0)
    for _ in range(3000):
        text = rng.integers(0, rng.integers(1, 6), rng.integers(0, 30)).tolist()
        nodes, length, match = (int(rng.integers(0, top)) for top in (10, 6, 5))
        assert draft.from_text(text, nodes=nodes, length=length, match=match) == _from_text(text, nodes, length, match)


@pytest.mark.parametrize(("vocab", "most"), [(1000000, 100), (300, 6000), (2, 1000)])
def test_a_draft_looks_only_where_the_last_token_recurs(vocab, most):
    """A long text in which little or nothing recurs: a draft is made for every call, and costs less than one."""
    text = _Counted(np.random.default_rng(vocab).integers(0, vocab, 100000).tolist())
    _Counted.asked[0] = 0
    draft.from_text(text)
    assert _Counted.asked[0] <= most


@pytest.mark.parametrize(("cache", "change"), [
    ({}, {"out": P + 16}), ({}, {"out": P, "q": P + 5 * 4 * 64 * 2 - 2}), ({}, {"q_stride": 4 * 64 + 8}),
    ({}, {"out": P + 4 * (4 * 64 + 8) * 2, "q_stride": 4 * 64 + 8}),
    ({"head_dim": 136, "slot_stride": 136, "head_stride": 16 * 136, "page_stride": 2 * 16 * 136}, {"q_stride": 4 * 136}),
])
def test_results_over_other_queries_are_refused(cache, change):
    _fails(_lib.lib().er_kv_tree(C.byref(_cache(**cache)), C.byref(_tree(**change)), None, 0, None), "share memory")


def test_lengths_over_what_a_compaction_reads_are_refused():
    """rows 3, lists of 4 by a stride of 5, at addresses of their own; lens_out over each in turn."""
    L, c = _lib.lib(), _cache()
    seqs, start, keep, counts = (P * i for i in (1, 2, 3, 4))
    for out in (seqs, start, start + 8, start - 8, keep, keep + 4 * 13, counts, counts - 4):
        _fails(L.er_kv_compact(C.byref(c), 2, 1 << 16, seqs, start, keep, 5, 4, counts, 3, out, None, None), "lens_out")
