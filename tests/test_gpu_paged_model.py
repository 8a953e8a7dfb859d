"""GPU: the decoder over a paged key-value cache (PagedKVCache): the
reference's logits and greedy tokens as with the contiguous cache, several
sequences in one call as each alone, page selection and eviction that leave
everything in as the full cache, and what a generation does under both."""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch
from conftest import golden
from golden.make_golden import MODEL_CASES, MODEL_NEW, MODEL_PROMPT
from kv_ref import choose, tokens

from expertrelay_b200 import _lib, synth
from expertrelay_b200.kv_cache import PagedKVCache
from expertrelay_b200.model import QwenMoeModel
from oracle.moe_oracle import rel_l2

pytestmark = pytest.mark.gpu

TOL = 1e-4  # the contiguous cache's, on the exact-fp32 expert path


def _model(case, cuda, path=_lib.PATH_GEMM):
    cfg, seed = MODEL_CASES[case]
    return QwenMoeModel(synth.make_model(cfg, seed=seed), device=cuda, path=path)


@pytest.mark.parametrize("case", range(len(MODEL_CASES)))
@pytest.mark.parametrize("options", [{}, {"page_size": 5}, {"mass": True, "page_size": 8}, {"select": (64, 1, 1), "page_size": 4}])
def test_paged_model_matches_reference(case, options, cuda):
    g = golden("model")
    model = _model(case, cuda)
    kv = model.new_paged_cache(1, MODEL_PROMPT + MODEL_NEW, **options)
    logits = model.forward(g[f"prompt{case}"], kv, all_logits=True).cpu().numpy()
    assert rel_l2(logits, g[f"prompt_logits{case}"]) < TOL
    tok = int(np.argmax(logits[-1]))
    for step in range(MODEL_NEW):
        assert tok == g[f"tokens{case}"][step]
        lg = model.forward([tok], kv).cpu().numpy()
        assert rel_l2(lg, g[f"step_logits{case}"][step]) < TOL
        tok = int(np.argmax(lg))
    if kv.mass is not None:
        # every row's weights sum to one for each query: length x queries a key head in all
        n, group = MODEL_PROMPT + MODEL_NEW, model.c.num_heads // model.c.num_kv_heads
        total = kv.mass.sum(-1).cpu().numpy()
        np.testing.assert_allclose(total, n * group, rtol=1e-4)
        assert torch.all(kv.mass[..., n:] == 0)
    kv.check()
    model.close()


def test_bf16_cache_is_near(cuda):
    """Keys and values rounded to 16 bits (2^-8 at most each) move the logits by about as much."""
    g = golden("model")
    model = _model(0, cuda)
    kv = model.new_paged_cache(1, MODEL_PROMPT, dtype=torch.bfloat16)
    logits = model.forward(g["prompt0"], kv, all_logits=True).cpu().numpy()
    assert rel_l2(logits, g["prompt_logits0"]) < 2.0 ** -5
    model.close()


def test_sequences_in_one_call_are_as_alone(cuda):
    model = _model(1, cuda)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, model.c.vocab_size, n) for n in (9, 1, 14)]
    alone = []
    for p in prompts:
        kv = model.new_cache(len(p) + 3)
        steps = [model.forward(p, kv).cpu().numpy()]
        for t in (5, 6, 7):
            steps.append(model.forward([t], kv).cpu().numpy())
        alone.append(steps)
    kv = model.new_paged_cache(4, 32, page_size=8)
    seqs = np.concatenate([np.full(len(p), s) for s, p in zip((0, 1, 3), prompts)])
    order = np.argsort(np.concatenate([np.arange(len(p)) for p in prompts]), kind="stable")  # interleaved
    logits = model.forward(np.concatenate(prompts)[order], kv, all_logits=True, seqs=seqs[order]).cpu().numpy()
    last = [int(np.flatnonzero(seqs[order] == s)[-1]) for s in (0, 1, 3)]
    for i in range(3):
        assert rel_l2(logits[last[i]], alone[i][0]) < TOL
    for j, t in enumerate((5, 6, 7)):
        lg = model.forward([t, t, t], kv, all_logits=True, seqs=[3, 0, 1]).cpu().numpy()
        for row, i in ((0, 2), (1, 0), (2, 1)):
            assert rel_l2(lg[row], alone[i][j + 1]) < TOL
    assert [kv.length(s) for s in range(4)] == [12, 4, 0, 17]
    kv.release(0)
    assert kv.length(0) == 0
    assert rel_l2(model.forward(prompts[0], kv).cpu().numpy(), alone[0][0]) < TOL
    kv.check()
    model.close()


def test_generation_with_eviction(cuda):
    model = _model(0, cuda)
    g = golden("model")
    kv = model.new_paged_cache(2, 64, page_size=4, mass=True)
    for s in (0, 1):
        model.forward(g["prompt0"], kv, seqs=[s] * MODEL_PROMPT)
    free = len(kv.pages.free)
    kv.evict(64, recent=8)  # nothing is that long
    assert len(kv.pages.free) == free and kv.length(0) == MODEL_PROMPT
    budget = MODEL_PROMPT - 3
    kv.evict(budget, sinks=1, recent=2)
    assert kv.length(0) == kv.length(1) == budget and int(kv.pages.position[0]) == MODEL_PROMPT
    assert len(kv.pages.free) >= free
    assert sorted(kv.pages.free + [int(p) for p in kv.pages.table.ravel() if p >= 0]) == list(range(32))
    tok = int(g["tokens0"][0])
    both = model.forward([tok, tok], kv, all_logits=True, seqs=[0, 1])
    assert torch.equal(both[0], both[1]) and torch.isfinite(both).all()
    assert kv.length(0) == budget + 1
    kv.check()
    model.close()


def test_paged_refusals(cuda):
    model = _model(0, cuda)
    kv = model.new_paged_cache(1, 8, page_size=4)
    with pytest.raises(ValueError, match="sequence length 9 exceeds the KV cache"):
        model.forward([1] * 9, kv)
    assert kv.length() == 0
    with pytest.raises(ValueError, match="outside"):
        model.forward([1], kv, seqs=[1])
    with pytest.raises(ValueError, match="one sequence for each"):
        model.forward([1, 2], kv, seqs=[0])
    with pytest.raises(ValueError, match="only with a PagedKVCache"):
        model.forward([1], model.new_cache(4), seqs=[0])
    with pytest.raises(ValueError, match="mass=True"):
        kv.evict(4)
    with pytest.raises(ValueError, match="mass and select"):
        model.new_paged_cache(1, 8, mass=True, select=(4, 1, 1))
    with pytest.raises(ValueError, match="select"):
        model.new_paged_cache(1, 8, select=(1, 1, 1))
    model.close()


def test_an_eviction_that_is_refused_changes_nothing(cuda):
    shape = SimpleNamespace(num_layers=1, num_kv_heads=1, head_dim=8)
    cache = PagedKVCache(shape, 1, 400000, page_size=100, pages=8, mass=True, device=cuda)  # more weights than are ranked
    cache.step([0] * 300)
    before = (cache.pages.table.copy(), sorted(cache.pages.free))
    with pytest.raises(ValueError, match="400000 weights"):
        cache.evict(200, recent=10)
    assert cache.length() == 300 and sorted(cache.pages.free) == before[1] and (cache.pages.table == before[0]).all()


class _Fails:
    """A model's MoE stack whose layer `at` raises on its next call."""

    def __init__(self, stack, at, error):
        self.stack, self.at, self.error = stack, at, error

    def moe(self, layer, *args, **kwargs):
        if layer == self.at and self.error is not None:
            error, self.error = self.error, None
            raise error
        return self.stack.moe(layer, *args, **kwargs)


@pytest.mark.parametrize("error", [RuntimeError("no room"), KeyboardInterrupt()])
@pytest.mark.parametrize("options", [{}, {"mass": True}, {"select": (2, 1, 1)}])
@pytest.mark.parametrize("at", [0, 1])
def test_a_call_that_raises_can_be_made_again(cuda, options, error, at):
    """Nothing of a call that fails between layers stays: lengths, positions, pages, weights; the same call again
    gives what it would have, prompts, steps of some sequences and steps of all."""
    g = golden("model")
    model = _model(0, cuda)
    kv, fresh = (model.new_paged_cache(3, 64, page_size=4, **options) for _ in range(2))
    prompt = [int(t) for t in g["prompt0"]]
    calls = [(prompt, [1] * len(prompt)), (prompt[:5] + prompt[:3], [2] * 5 + [0] * 3), ([7, 8], [1, 2]), ([3, 4, 5], [0, 1, 2]),
             ([9] * 6, [0, 1, 2] * 2)]
    stack = model.stack
    for tokens, seqs in calls:
        before = (kv.pages.table.copy(), kv.pages.length.copy(), kv.pages.position.copy(), list(kv.pages.free),
                  None if kv.mass is None else kv.mass.clone())
        model.stack = _Fails(stack, at, error)
        with pytest.raises(type(error)):
            model.forward(tokens, kv, seqs=seqs)
        model.stack = stack
        assert (kv.pages.table == before[0]).all() and (kv.table.cpu().numpy() == before[0]).all()
        assert (kv.pages.length == before[1]).all() and (kv.pages.position == before[2]).all()
        assert kv.pages.free == before[3] and (kv.mass is None or torch.equal(kv.mass, before[4]))
        got, want = (model.forward(tokens, c, all_logits=True, seqs=seqs) for c in (kv, fresh))
        assert torch.equal(got, want)
    assert kv.mass is None or torch.equal(kv.mass, fresh.mass)
    with pytest.raises(ValueError, match="token ids"):
        model.forward([model.c.vocab_size], kv, seqs=[1])
    assert torch.equal(model.forward([2], kv, seqs=[1]), model.forward([2], fresh, seqs=[1]))
    kv.check()
    model.close()


def test_only_the_last_step_is_taken_back(cuda):
    shape = SimpleNamespace(num_layers=1, num_kv_heads=1, head_dim=8)
    cache = PagedKVCache(shape, 2, 16, page_size=4, device=cuda)
    first, second = cache.step([0] * 5), cache.step([1])
    with pytest.raises(ValueError, match="last step"):
        cache.undo(first)
    cache.undo(second)
    with pytest.raises(ValueError, match="last step"):
        cache.undo(second)
    third = cache.step([1, 1])
    cache.release(1)
    with pytest.raises(ValueError, match="last step"):
        cache.undo(third)
    assert cache.length(0) == 5 and cache.length(1) == 0 and len(cache.pages.free) == 6


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize(("budget", "sinks", "recent"), [(32, 4, 8), (13, 0, 1), (61, 2, 5), (63, 0, 0)])
@pytest.mark.parametrize("pages", [None, 34, 40, 64])
def test_eviction_whatever_pages_are_free(cuda, dtype, budget, sinks, recent, pages):
    """Pools without a free page, with one sequence's worth, with all: the same places stay, in pages of the pool, and
    later calls go on from them."""
    shape = SimpleNamespace(num_layers=2, num_kv_heads=2, head_dim=16)
    lens = [64, 64, 5, 64, 50]
    cache = PagedKVCache(shape, 5, 64, page_size=8, pages=pages or 32, dtype=dtype, mass=True, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(budget)
    seqs = [s for s, n in enumerate(lens) for _ in range(n)]
    step = cache.step(seqs)
    for layer in range(2):
        cache.attend(layer, step, torch.randn((len(seqs), 6 * 16), generator=gen, device=cuda), 2, 1e4)
    if pages is None:
        assert not cache.pages.free
    table = torch.from_numpy(cache.pages.table.copy())
    old = {(i, s): (tokens(cache.k[i], table, s, n), tokens(cache.v[i], table, s, n)) for i in range(2) for s, n in enumerate(lens)}
    mass = cache.mass.cpu().numpy()
    cache.evict(budget, sinks=sinks, recent=recent)
    cache.check()
    total = pages or 32
    used = [int(p) for p in cache.pages.table.ravel() if p >= 0]
    assert sorted(used + cache.pages.free) == list(range(total)) and len(set(used)) == len(used)
    assert (cache.table.cpu().numpy() == cache.pages.table).all()
    assert cache.pages.position.tolist() == lens
    table = torch.from_numpy(cache.pages.table.copy())
    for s, n in enumerate(lens):
        m = min(n, budget)
        assert cache.length(s) == m
        for i in range(2):
            k, v = tokens(cache.k[i], table, s, m), tokens(cache.v[i], table, s, m)
            for h in range(2):
                ids = choose(mass[i, s, h], n, budget, sinks, recent)
                assert np.array_equal(k[h], old[i, s][0][h][ids]) and np.array_equal(v[h], old[i, s][1][h][ids])
                assert np.array_equal(cache.mass[i, s, h].cpu().numpy(), np.pad(mass[i, s, h][ids], (0, 64 - m)))
    step = cache.step([0, 1, 2, 3, 4])
    for layer in range(2):
        assert torch.isfinite(cache.attend(layer, step, torch.randn((5, 96), generator=gen, device=cuda), 2, 1e4)).all()
    cache.check()


def test_an_eviction_that_fails_between_layers_changes_nothing(cuda, monkeypatch):
    from expertrelay_b200 import kv as operators

    shape = SimpleNamespace(num_layers=2, num_kv_heads=1, head_dim=8)
    for pages in (8, 16):  # without free pages, and with some
        cache = PagedKVCache(shape, 2, 32, page_size=8, pages=pages, mass=True, device=cuda)
        step = cache.step([0] * 32 + [1] * 32)
        for layer in range(2):
            cache.attend(layer, step, torch.randn((64, 3 * 8), device=cuda), 1, 1e4)
        before = [x.clone() for x in (cache.k, cache.v, cache.mass, cache.table)]
        host = (cache.pages.table.copy(), cache.pages.length.copy(), list(cache.pages.free))
        real, calls = operators.evict, []

        def failing(*args, **kwargs):
            calls.append(0)
            if len(calls) == 2:
                raise RuntimeError("no room")
            return real(*args, **kwargs)

        monkeypatch.setattr(operators, "evict", failing)
        with pytest.raises(RuntimeError, match="no room"):
            cache.evict(20, recent=4)
        monkeypatch.setattr(operators, "evict", real)
        assert (cache.pages.table == host[0]).all() and (cache.pages.length == host[1]).all() and cache.pages.free == host[2]
        assert torch.equal(cache.mass, before[2]) and torch.equal(cache.table, before[3])
        table = torch.from_numpy(host[0])
        for s in (0, 1):
            for i in range(2):
                assert np.array_equal(tokens(cache.k[i], table, s, 32), tokens(before[0][i], table, s, 32))
                assert np.array_equal(tokens(cache.v[i], table, s, 32), tokens(before[1][i], table, s, 32))


def test_a_sequence_outside_the_cache_is_not_another_one(cuda):
    cache = PagedKVCache(SimpleNamespace(num_layers=1, num_kv_heads=1, head_dim=8), 2, 16, page_size=4, mass=True, device=cuda)
    cache.step([1] * 5)
    cache.mass[:, 1] = 1
    for call in (lambda: cache.release(-1), lambda: cache.release(2), lambda: cache.length(-1), lambda: cache.length(2)):
        with pytest.raises(ValueError, match="outside"):
            call()
    assert cache.length(1) == 5 and (cache.mass[:, 1] == 1).all()
