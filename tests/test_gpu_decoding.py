"""GPU: several continuations of a text at once, all of it together: trees of
drafted tokens through the decoder, accepted paths, forks and beams over
shared pages, against the same texts alone and against greedy decoding."""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch
from conftest import golden
from golden.make_golden import MODEL_CASES, MODEL_NEW
from kv_ref import tokens

from expertrelay_b200 import _lib, draft, kv, synth
from expertrelay_b200.kv_cache import PagedKVCache
from expertrelay_b200.model import QwenMoeModel
from oracle.moe_oracle import rel_l2

pytestmark = pytest.mark.gpu

TOL = 1e-4  # the paged cache's against the reference
PARENTS = [-1, 0, 0, 1, -1, 4, 2, 6, 7, 4]


def _model(case, cuda):
    cfg, seed = MODEL_CASES[case]
    return QwenMoeModel(synth.make_model(cfg, seed=seed), device=cuda, path=_lib.PATH_GEMM)


def _path(node, parents=PARENTS):
    path = []
    while node >= 0:
        path.insert(0, node)
        node = parents[node]
    return path


def _whole(kv):
    """Every page is free or as often used as tables name it, and no sequence's next place lies in a shared one."""
    named = np.bincount(kv.pages.table[kv.pages.table >= 0], minlength=len(kv.pages.uses))
    assert (named == kv.pages.uses).all() and sorted(kv.pages.free) == np.flatnonzero(named == 0).tolist()
    assert (kv.table.cpu().numpy() == kv.pages.table).all()
    for s in range(kv.seqs):
        full, part = divmod(kv.length(s), kv.page_size)
        assert not part or kv.pages.uses[kv.pages.table[s, full]] == 1


@pytest.mark.parametrize("case", range(len(MODEL_CASES)))
@pytest.mark.parametrize("options", [{}, {"page_size": 5}, {"select": (64, 1, 1), "page_size": 4}, {"dtype": torch.bfloat16}])
def test_drafted_tokens_are_as_their_paths_alone(case, options, cuda):
    g = golden("model")
    model = _model(case, cuda)
    tol = 2.0 ** -5 if "dtype" in options else TOL  # keys and values may round the other way
    prompts = [[int(t) for t in g[f"prompt{case}"]], [3, 1, 2]]
    rng = np.random.default_rng(case)
    drafted = [rng.integers(0, model.c.vocab_size, len(PARENTS)).tolist(), [5]]
    parents = [PARENTS, [-1]]
    kv = model.new_paged_cache(3, 64, **options)
    for s, p in zip((2, 0), prompts):
        model.forward(p, kv, seqs=[s] * len(p))
    seqs = [2] * len(PARENTS) + [0]
    logits = model.forward(sum(drafted, []), kv, all_logits=True, seqs=seqs, parents=sum(parents, [])).cpu().numpy()
    for t, prompt in enumerate(prompts):
        for node in range(len(parents[t])):
            text = prompt + [drafted[t][i] for i in _path(node, parents[t])]
            want = model.forward(text, model.new_paged_cache(1, 64, **options)).cpu().numpy()
            assert rel_l2(logits[node if t == 0 else len(PARENTS)], want) < tol
    with pytest.raises(ValueError, match="neither accepted"):
        model.forward([1], kv)
    paths = [_path(8), []]  # 0 2 6 7 8
    kv.accept(kv.drafted, paths)
    assert kv.drafted is None and kv.length(2) == len(prompts[0]) + 5 and kv.length(0) == 3
    assert int(kv.pages.position[2]) == kv.length(2)
    _whole(kv)
    text = prompts[0] + [drafted[0][i] for i in paths[0]]
    for t in (4, 9, 11):  # and on from there
        text.append(t)
        got = model.forward([t, t], kv, all_logits=True, seqs=[2, 0])[0].cpu().numpy()
        want = model.forward(text, model.new_paged_cache(1, 64, **options)).cpu().numpy()
        assert rel_l2(got, want) < tol
    kv.check()
    model.close()


@pytest.mark.parametrize("case", range(len(MODEL_CASES)))
@pytest.mark.parametrize("options", [{}, {"page_size": 3}, {"select": (64, 1, 1), "page_size": 4}])
def test_drafted_generation_is_greedy_generation(case, options, cuda):
    g = golden("model")
    model = _model(case, cuda)
    prompt, want = [int(t) for t in g[f"prompt{case}"]], [int(t) for t in g[f"tokens{case}"]]
    new = len(want)

    def knows(text):  # the answer, beside others
        rest = want[len(text) - len(prompt):]
        return [0, 1, *rest[:4]], [-1, 0, *([-1, 2, 3, 4][:len(rest)])]

    def wrong(text):
        return [(text[-1] + i) % model.c.vocab_size for i in range(3)], [-1, 0, 1]

    calls = {}
    for name, d in (("text", draft.from_text), ("knows", knows), ("wrong", wrong), ("none", lambda text: ([], []))):
        kv = model.new_paged_cache(2, 64, **options)
        out, calls[name] = model.generate_drafted(prompt, new, d, kv=kv, seq=1)
        assert out == want
        assert kv.length(1) == len(prompt) + new - 1 and kv.length(0) == 0
        _whole(kv)
        kv.check()
    assert calls["none"] == new - 1 and calls["knows"] == -(-(new - 1) // 5)
    assert model.generate_drafted(prompt, 1)[0] == want[:1]
    tight = model.new_paged_cache(1, len(prompt) + new - 1, page_size=1)  # no room for many guesses
    assert model.generate_drafted(prompt, new, knows, kv=tight)[0] == want
    model.close()


@pytest.mark.parametrize("options", [{}, {"page_size": 4, "select": (64, 1, 1)}, {"page_size": 5, "mass": True}])
def test_texts_that_go_on_from_shared_pages(options, cuda):
    model = _model(1, cuda)
    prompt = [int(t) for t in golden("model")["prompt1"]]
    kv = model.new_paged_cache(4, 32, **options)
    model.forward(prompt, kv)
    kv.reorder([1, 2], [0, 0])
    _whole(kv)
    full = len(prompt) // kv.page_size
    assert (kv.pages.table[:3, :full] == kv.pages.table[0, :full]).all()
    texts = [list(prompt) for _ in range(3)] + [[]]
    for step, order in enumerate(([0, 1, 2, 3], [1, 1, 0, 3], [2, 2, 2, 2], [3, 0, 1, 3])):
        for s in range(4):
            texts[s].append((3 * s + step) % model.c.vocab_size)
        got = model.forward([t[-1] for t in texts], kv, all_logits=True, seqs=[0, 1, 2, 3]).cpu().numpy()
        for s in range(4):
            want = model.forward(texts[s], model.new_paged_cache(1, 32, **options)).cpu().numpy()
            assert rel_l2(got[s], want) < TOL
        kv.reorder([0, 1, 2, 3], order)
        _whole(kv)
        texts = [list(texts[p]) for p in order]
        assert [kv.length(s) for s in range(4)] == [len(t) for t in texts]
    if kv.mass is not None:
        kv.evict(6, sinks=1, recent=2)
        _whole(kv)
        assert max(kv.length(s) for s in range(4)) <= 6
        assert torch.isfinite(model.forward([1, 2, 3, 4], kv, all_logits=True, seqs=[0, 1, 2, 3])).all()
    for s in range(4):
        kv.release(s)
    assert sorted(kv.pages.free) == list(range(len(kv.pages.uses)))
    kv.check()
    model.close()


def test_bounds_follow_accepted_drafts_and_forks(cuda):
    """Rejected drafts leave nothing in the bounds that page choices go by: after each step that appends, they are those
    of the keys that are there."""
    shape = SimpleNamespace(num_layers=2, num_kv_heads=2, head_dim=16)
    cache = PagedKVCache(shape, 3, 40, page_size=4, select=(3, 1, 1), device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(1)

    def run(seqs, parents=None, loud=1.0):
        step = cache.step(seqs, parents)
        for layer in range(2):
            qkv = torch.randn((len(seqs), 6 * 16), generator=gen, device=cuda)
            cache.attend(layer, step, qkv * loud, 2, 1e4)
        return step

    def right():
        lens = torch.tensor(cache.pages.length, dtype=torch.int32, device=cuda)
        for layer in range(2):
            fresh = kv.PageBounds.new(cache.layers[layer])
            kv.page_bounds(cache.layers[layer], fresh, lens, torch.zeros_like(lens))
            used = [int(p) for s in range(3) for p in cache.pages.table[s, :-(-cache.length(s) // 4)]]
            assert torch.equal(fresh.codes[used], cache.bounds[layer].codes[used])
            assert torch.equal(fresh.scales[used], cache.bounds[layer].scales[used])

    run([0] * 9 + [1] * 3)
    right()
    step = run([0] * 8 + [1] * 2, [-1, 0, 1, 0, 3, 4, 5, 2, -1, -1], loud=50.0)
    cache.accept(step, [[0, 3, 4, 5, 6], [1]])
    right()
    cache.undo(run([0] * 4, [-1] * 4, loud=500.0))
    right()
    cache.accept(run([1] * 4, [-1] * 4, loud=500.0), [[]])
    right()
    cache.reorder([2], [0])
    run([0, 1, 2])
    right()
    cache.reorder([0, 1, 2], [2, 2, 0])
    run([2, 1, 0])
    right()
    cache.check()


@pytest.mark.parametrize("at", [0, 1])
def test_drafted_calls_that_raise_can_be_made_again(at, cuda):
    """Nothing stays of a call that fails between layers, and a draft of tokens that there are none of is refused."""
    model = _model(0, cuda)
    kv, fresh = (model.new_paged_cache(2, 32, page_size=4) for _ in range(2))
    for c in (kv, fresh):
        model.forward([1, 2, 3, 4, 5], c, seqs=[1] * 5)
    before = (kv.pages.table.copy(), kv.pages.length.copy(), kv.pages.position.copy(), list(kv.pages.free))
    stack = model.stack

    class Fails:
        def moe(self, layer, *args, **kwargs):
            if layer == at:
                raise RuntimeError("no room")
            return stack.moe(layer, *args, **kwargs)

    for tokens, error in (([7, 8, 9], RuntimeError), ([7, model.c.vocab_size, 9], ValueError)):
        model.stack = Fails() if error is RuntimeError else stack
        with pytest.raises(error):
            model.forward(tokens, kv, all_logits=True, seqs=[1] * 3, parents=[-1, 0, 0])
        model.stack = stack
        assert kv.drafted is None and (kv.pages.table == before[0]).all() and (kv.pages.length == before[1]).all()
        assert (kv.pages.position == before[2]).all() and kv.pages.free == before[3]
    got, want = (model.forward([7, 8, 9], c, all_logits=True, seqs=[1] * 3, parents=[-1, 0, 0]) for c in (kv, fresh))
    assert torch.equal(got, want)
    model.close()


@pytest.mark.parametrize("pages", [8, 9, 14])
def test_eviction_leaves_shared_pages_alone(pages, cuda):
    """A sequence that shares its first pages is cut into others; the one it shares them with reads what it read."""
    shape = SimpleNamespace(num_layers=2, num_kv_heads=2, head_dim=16)
    cache = PagedKVCache(shape, 3, 48, page_size=8, pages=pages, mass=True, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(pages)

    def run(seqs):
        step = cache.step(seqs)
        for layer in range(2):
            cache.attend(layer, step, torch.randn((len(seqs), 6 * 16), generator=gen, device=cuda), 2, 1e4)

    run([0] * 28)
    cache.reorder([2], [0])
    _whole(cache)
    run([2] * 20)  # 48 places: 3 pages shared, 3 of its own
    assert len(cache.pages.free) == pages - 7
    table = torch.from_numpy(cache.pages.table.copy())
    old = [tokens(pool[i], table, 0, 28) for i in range(2) for pool in (cache.k, cache.v)]
    cache.evict(30, recent=4)  # 4 pages
    _whole(cache)
    assert [cache.length(s) for s in range(3)] == [28, 0, 30]
    table = torch.from_numpy(cache.pages.table.copy())
    for a, b in zip(old, [tokens(pool[i], table, 0, 28) for i in range(2) for pool in (cache.k, cache.v)]):
        assert np.array_equal(a, b)
    cache.check()


def test_eviction_without_pages_of_its_own(cuda):
    shape = SimpleNamespace(num_layers=1, num_kv_heads=1, head_dim=8)
    cache = PagedKVCache(shape, 2, 32, page_size=8, pages=4, mass=True, device=cuda)
    step = cache.step([0] * 32)
    cache.attend(0, step, torch.randn((32, 3 * 8), device=cuda), 1, 1e4)
    cache.reorder([1], [0])
    with pytest.raises(ValueError, match="out of pages"):
        cache.evict(20, recent=4)
    _whole(cache)
    assert cache.length(0) == cache.length(1) == 32


@pytest.mark.parametrize("case", range(len(MODEL_CASES)))
@pytest.mark.parametrize(("beams", "end"), [(1, None), (3, None), (5, 7), (8, None)])
def test_beam_search_finds_what_a_plain_one_does(case, beams, end, cuda):
    g = golden("model")
    model = _model(case, cuda)
    prompt, new = [int(t) for t in g[f"prompt{case}"]], 5
    kv = model.new_paged_cache(beams, 64, page_size=3)
    got = model.beam_search(prompt, beams, new, end=end, kv=kv)
    _whole(kv)
    kv.check()

    def after(text):
        return torch.log_softmax(model.forward(prompt + text, model.new_cache(64)).double(), 0).cpu()

    live, done = [([], 0.0)], []
    for n in range(new):
        every = sorted(((v + float(p), t + [i]) for t, v in live for i, p in enumerate(after(t))), reverse=True)
        every = every[:beams if end is None else 2 * beams]
        done += [(t, v) for v, t in every if t[-1] == end or n + 1 == new]
        live = [(t, v) for v, t in every if t[-1] != end][:beams]
    done = sorted(done, key=lambda d: -d[1])[:beams]
    assert [t for t, _ in got] == [t for t, _ in done]
    np.testing.assert_allclose([v for _, v in got], [v for _, v in done], rtol=1e-4)
    if beams == 1:
        assert got[0][0][:MODEL_NEW] == [int(t) for t in g[f"tokens{case}"]][:MODEL_NEW]
    model.close()


def test_decoding_refusals(cuda):
    model = _model(0, cuda)
    kv = model.new_paged_cache(2, 16, page_size=4)
    model.forward([1, 2, 3], kv)
    before = (kv.pages.table.copy(), kv.length(0))
    for parents, seqs, words in [([-1, 1], [0, 0], "before the child"), ([-1, -2], [0, 0], "before the child"), ([0], [0], "before the child"),
                                 ([-1], [0, 0], "one for each"), ([-1, -1, -1], [0, 1, 0], "in one run"), ([], [], "one for each"),
                                 ([-1] * 14, [0] * 14, "exceeds the KV cache")]:
        with pytest.raises(ValueError, match=words):
            model.forward([1] * len(seqs), kv, seqs=seqs, parents=parents)
        assert (kv.pages.table == before[0]).all() and kv.length(0) == before[1] and kv.drafted is None
    with pytest.raises(ValueError, match="at most 4096 of 256"):
        kv.step([0] * 257, [-1] * 257)
    with pytest.raises(ValueError, match="only with a PagedKVCache"):
        model.forward([1], model.new_cache(4), parents=[-1])
    with pytest.raises(ValueError, match="mass=True"):
        model.new_paged_cache(1, 8, mass=True).step([0], [-1])
    logits = model.forward([4, 5, 6], kv, all_logits=True, seqs=[0] * 3, parents=[-1, 0, -1])
    step = kv.drafted
    for paths in ([[1]], [[0, 2]], [[0, 0]], [[3]], [[-1]], [], [[0], [1]]):
        with pytest.raises(ValueError, match="accept"):
            kv.accept(step, paths)
    for call in (lambda: kv.step([0]), lambda: kv.reorder([1], [0]), lambda: kv.release(0)):
        with pytest.raises(ValueError, match="neither accepted"):
            call()
    kv.undo(step)
    with pytest.raises(ValueError, match="not the cache's last step"):
        kv.accept(step, [[0]])
    assert (kv.pages.table == before[0]).all() and kv.length(0) == before[1]
    assert torch.equal(logits, model.forward([4, 5, 6], kv, all_logits=True, seqs=[0] * 3, parents=[-1, 0, -1]))
    kv.accept(kv.drafted, [[]])
    assert kv.length(0) == before[1]
    for seqs, parents, words in [([0, 0], [1, 1], "distinct"), ([0], [0, 1], "distinct"), ([2], [0], "outside"), ([0], [-1], "outside")]:
        with pytest.raises(ValueError, match=words):
            kv.reorder(seqs, parents)
    with pytest.raises(ValueError, match="at least"):
        model.beam_search([1], 0, 3)
    with pytest.raises(ValueError, match="at most 64"):
        model.beam_search([1], 65, 3, end=0)
    with pytest.raises(ValueError, match="at least 1"):
        model.generate_drafted([1], 0)
    model.close()


def test_a_call_that_the_device_found_wrong_ends_the_decoding(cuda):
    """Attention that gave up waiting, or met a bad page: no token comes of it, and the draft's places are given back."""
    model = _model(0, cuda)
    prompt = [1, 2, 3, 4, 5]
    want = model.generate(prompt, 4)[0]
    kv = model.new_paged_cache(2, 32, page_size=4)

    def spoils(text):
        kv.status.fill_(_lib.KV_GAVE_UP)
        return [7, 8], [-1, 0]

    with pytest.raises(RuntimeError, match="gave up"):
        model.generate_drafted(prompt, 4, spoils, kv=kv)
    assert kv.drafted is None and kv.length(0) == len(prompt)
    _whole(kv)
    kv.release(0)
    assert model.generate_drafted(prompt, 4, lambda text: ([7, 8], [-1, 0]), kv=kv)[0] == want
    kv.release(0)
    for bit, error in ((_lib.KV_GAVE_UP, RuntimeError), (_lib.KV_BAD_PAGE, ValueError)):
        kv.status.fill_(bit)
        with pytest.raises(error, match="paged cache"):
            model.beam_search(prompt, 2, 4, kv=kv)
        for s in range(2):
            kv.release(s)
    assert model.beam_search(prompt, 1, 4, kv=kv)[0][0] == want
    model.close()


def test_searches_go_on_from_what_the_cache_holds(cuda):
    """A text in two parts gives what it gives in one, and no sequence's text is written over."""
    model = _model(1, cuda)
    text = [3, 1, 4, 1, 5, 9, 2, 6]
    want = model.generate(text, 5)[0]

    def fresh(**options):
        kv = model.new_paged_cache(4, 32, page_size=4, **options)
        model.forward(text[:5], kv, seqs=[0] * 5)
        return kv

    kv = fresh()
    assert model.generate_drafted(text[5:], 5, lambda t: ([want[0], 7], [-1, 0]), kv=kv)[0] == want
    assert kv.length(0) == len(text) + 4
    kv = fresh()
    assert model.beam_search(text[5:], 1, 5, kv=kv)[0][0] == want
    one, two = model.beam_search(text, 3, 5), model.beam_search(text[5:], 3, 5, kv=fresh())
    assert [t for t, _ in one] == [t for t, _ in two]
    np.testing.assert_allclose([v for _, v in one], [v for _, v in two], rtol=1e-4)
    for s in (1, 2):
        kv = fresh()
        model.forward([7, 7], kv, seqs=[s, s])
        before = (kv.pages.table.copy(), kv.pages.length.copy())
        with pytest.raises(ValueError, match="not empty"):
            model.beam_search(text[5:], 3, 5, kv=kv)
        assert (kv.pages.table == before[0]).all() and (kv.pages.length == before[1]).all()
    kv = fresh(mass=True)
    with pytest.raises(ValueError, match="mass=True"):
        model.generate_drafted(text[5:], 5, kv=kv)
    assert kv.length(0) == 5
    model.close()
