"""GPU: beam search's selection against its definition (tests/tree_ref.py)."""

from __future__ import annotations

import numpy as np
import pytest
import torch
from tree_ref import beam_reference

from expertrelay_b200 import beam

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
INF = float("inf")


def _check(logits, scores, count, got):
    batch, beams = scores.shape
    want = beam_reference(logits.double().cpu().numpy().reshape(batch, beams, -1), scores.double().cpu().numpy(), count)
    value, which, token = (x.cpu().numpy() for x in got)
    assert value.dtype == np.float32 and which.dtype == token.dtype == np.int32
    for b in range(batch):
        assert [(int(w), int(t)) for w, t in zip(which[b], token[b])] == [(w, t) for _, w, t in want[b]], f"batch {b}"
        v = np.array([x[0] for x in want[b]])
        fine = np.isfinite(v)
        assert np.array_equal(value[b][~fine], v[~fine])
        # the log-sum is a 64-bit sum of 32-bit exponentials, each within 2^-22 (two units) and 2^-24 times its
        # argument of the formula: together under 2^-21, then a rounding of the result
        assert np.all(np.abs(value[b][fine] - v[fine]) <= 2.0 ** -21 + 2.0 ** -24 * np.abs(v[fine]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize(("batch", "beams", "vocab", "count"), [
    (1, 1, 1, 1), (1, 4, 151936, 8), (3, 5, 50257, 10), (2, 8, 4097, 128), (7, 3, 33, 99), (1, 1, 128, 128), (2, 1, 4095, 2),
    (1, 300, 129, 64), (5, 2, 12289, 77), (70, 6, 300, 12), (1, 2, 1000003, 4),
])
def test_select_matches_the_definition(cuda, dtype, batch, beams, vocab, count):
    gen = torch.Generator(device="cuda").manual_seed(vocab + count)
    logits = (torch.randn((batch * beams, vocab), generator=gen, device="cuda") * 3).to(dtype)
    scores = -5 * torch.rand((batch, beams), generator=gen, device="cuda")
    got = beam.select(logits, scores, count)
    _check(logits, scores, count, got)
    again = beam.select(logits, scores, count)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [37, 5000, 20001])
def test_ties_masks_and_beams_that_offer_nothing(cuda, dtype, vocab):
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    # few values, so that ties cross the parts, the threads and the beams; the beams of a batch are alike
    row = torch.randint(0, 3, (vocab,), generator=gen, device="cuda").to(dtype)
    for logits in (row.expand(6, vocab).contiguous(), torch.zeros((6, vocab), dtype=dtype, device="cuda"),
                   torch.arange(vocab, device="cuda").to(dtype).expand(6, vocab).contiguous(),
                   torch.arange(vocab, 0, -1, device="cuda").to(dtype).expand(6, vocab).contiguous()):
        _check(logits, torch.zeros((2, 3), device="cuda"), 20, beam.select(logits, torch.zeros((2, 3), device="cuda"), 20))
        scores = torch.tensor([[0.0, -INF, -INF], [-INF, 0.0, float("nan")]], device="cuda")
        _check(logits, scores, 20, beam.select(logits, scores, 20))
    # what a grammar leaves: two tokens, then -inf ones in order; rows without any, with NaN or +inf among them
    logits = torch.full((6, vocab), -INF, device="cuda").to(dtype)
    logits[0, 5], logits[0, vocab - 1], logits[2, 1] = 1.0, 2.0, -30.0
    logits[3], logits[4], logits[5] = 0.5, 0.25, 0.125
    logits[4, vocab // 2], logits[5, vocab - 1] = float("nan"), INF
    scores = torch.tensor([[-1.0, -2.0, -3.0], [-90.0, 0.0, 0.0]], device="cuda")
    _check(logits, scores, 16, beam.select(logits, scores, 16))
    scores = torch.tensor([[-INF, -INF, -INF], [INF, -INF, -3.4e38]], device="cuda")
    _check(logits, scores, 16, beam.select(logits, scores, 16))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_equal_rows_on_any_alignment_tie(cuda, dtype):
    """Beams with the same logits and score tie exactly, wherever their rows begin."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    row = (torch.randn((50257,), generator=gen, device="cuda") * 2).to(dtype)
    wide = torch.empty((4, 50261 + 8), dtype=dtype, device="cuda")
    logits = wide[:, 3:3 + 50257]
    logits.copy_(row)
    scores = torch.full((1, 4), -1.5, device="cuda")
    got = beam.select(logits, scores, 12)
    _check(logits, scores, 12, got)
    assert got[1][0].tolist() == [0, 1, 2, 3] * 3


def test_far_and_close_values(cuda):
    """Values of different beams that 32 bits cannot tell apart, and logits far from zero."""
    logits = torch.full((2, 300), -60.0, device="cuda")
    logits[0, 7] = logits[1, 9] = 80.0
    scores = torch.tensor([[-1.0e7, -1.0e7]], device="cuda")
    logits[1, 10] = 63.0  # beam 1's best is a little under beam 0's
    _check(logits, scores, 4, beam.select(logits, scores, 4))
    logits = torch.randn((4, 4000), device="cuda") + 1.0e4
    _check(logits, torch.zeros((1, 4), device="cuda"), 30, beam.select(logits, torch.zeros((1, 4), device="cuda"), 30))


def test_captured_and_on_another_stream(cuda):
    gen = torch.Generator(device="cuda").manual_seed(5)
    logits, scores = torch.randn((8, 9000), generator=gen, device="cuda"), torch.zeros((2, 4), device="cuda")
    beam.select(logits, scores, 6)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(beam.select(logits, scores, 6))
        graphs.append(g)
    for _ in range(3):
        logits.copy_(torch.randn((8, 9000), generator=gen, device="cuda"))
        for g, out in zip(graphs, outs):
            g.replay()
            _check(logits, scores, 6, out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = beam.select(logits, scores, 6)
    side.synchronize()
    _check(logits, scores, 6, got)


def test_refusals(cuda):
    x, s = torch.zeros((6, 50), device="cuda"), torch.zeros((2, 3), device="cuda")
    for call, words in ((lambda: beam.select(x.half(), s, 4), "logits"), (lambda: beam.select(x.cpu(), s, 4), "logits"),
                        (lambda: beam.select(x[0], s, 4), "logits"), (lambda: beam.select(x.T, s, 4), "logits"),
                        (lambda: beam.select(x[:5], s, 4), "rows"), (lambda: beam.select(x, s.double(), 4), "scores"),
                        (lambda: beam.select(x, s[0], 4), "scores"), (lambda: beam.select(x, s.cpu(), 4), "scores"),
                        (lambda: beam.select(x, s, 0), "count"), (lambda: beam.select(x, s, -3), "count"),
                        (lambda: beam.select(x, s, 129), "count"), (lambda: beam.select(x[:, :2], s, 7), "count"),
                        (lambda: beam.select(x[:1].expand(6, 50), s, 4), "stride"),
                        (lambda: beam.select(x, s, 4, workspace=torch.empty(8, device="cuda")), "workspace"),
                        (lambda: beam.select(torch.zeros((1025, 4), device="cuda"), torch.zeros((1, 1025), device="cuda"), 4), "beams"),
                        (lambda: beam.select(torch.zeros((65536, 1), device="cuda"), torch.zeros((65536, 1), device="cuda"), 1), "rows")):
        with pytest.raises(ValueError, match=words):
            call()
    assert [tuple(t.shape) for t in beam.select(x[:0], s[:0], 4)] == [(0, 4)] * 3


def test_rows_that_rise_with_every_tile(cuda):
    """Log-sums to the bound that _check states wherever a row's greatest come: every tile of 4096 here has a new
    maximum, a little above the last one. The scores make the values near zero, so that no rounding hides the sum's."""
    rows, vocab = 600, 500003
    up = torch.linspace(2e-4, 0.08, rows, dtype=torch.float64, device="cuda")
    tile = torch.arange(vocab, device="cuda") // 4096
    logits = torch.empty((rows, vocab), device="cuda")
    want, scores = [], []
    for r in range(0, rows, 100):
        logits[r:r + 100] = (up[r:r + 100, None] * tile).float()
        x = logits[r:r + 100].double()
        lse = torch.logsumexp(x, -1)
        scores.append((lse - x[:, -1]).float())
        want.append(scores[-1].double() + (x[:, -1] - lse))
    want, scores = torch.cat(want), torch.cat(scores)
    got, beams, tokens = beam.select(logits, scores[:, None], 1)
    assert torch.all(beams == 0) and torch.all(tokens[:, 0] == int(torch.nonzero(tile == tile[-1])[0]))
    off = (got[:, 0].double() - want).abs().max().item()
    assert off <= 2.0 ** -21, f"{off * 2 ** 21:.3g} of the bound"


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize(("beams", "vocab", "count"), [(1, 5000, 20), (3, 5000, 128), (4, 5, 17), (300, 9, 100), (2, 30011, 1)])
def test_within_a_beam_the_higher_logit_wins(cuda, dtype, beams, vocab, count):
    """Scores so far from zero that 64 bits hold no difference of the logits: all values of beams of one score are equal,
    and the lower beam's come first, by logit, then token."""
    gen = torch.Generator(device="cuda").manual_seed(vocab + beams)
    logits = (torch.randn((2 * beams, vocab), generator=gen, device="cuda") * 3).to(dtype)
    scores = torch.full((2, beams), -1.0e20, device="cuda")
    if beams > 1:
        scores[1, 0] = -2.0e20  # behind all others
    value, which, token = beam.select(logits, scores, count)
    for b, order in enumerate((list(range(beams)), [*range(1, beams), 0])):
        want = []
        for i in order:
            row = logits[b * beams + i].double()
            want += [(i, int(t)) for t in torch.sort(row, descending=True, stable=True).indices[:count]]
        assert list(zip(which[b].tolist(), token[b].tolist())) == want[:count]
        assert torch.equal(value[b], scores[b][which[b].long()])


def test_the_longest_rows(cuda):
    """The last part of a row that ends 65536 short of 2^31."""
    vocab = 0x7fff0000
    logits = torch.full((1, vocab), -INF, dtype=BF16, device="cuda")
    at = {vocab - 1: 2.0, 3: 1.0, vocab - 4097: 1.5, vocab - 2000000: -1.0}
    for token, x in at.items():
        logits[0, token] = x
    value, _, token = beam.select(logits, torch.zeros((1, 1), device="cuda"), 4)
    assert token[0].tolist() == sorted(at, key=at.get, reverse=True)
    x = torch.tensor(sorted(at.values(), reverse=True), dtype=torch.float64)
    torch.testing.assert_close(value[0].cpu().double(), x - torch.logsumexp(x, 0), rtol=0, atol=2.0 ** -20)
    with pytest.raises(ValueError, match="vocabulary"):
        beam.select(torch.empty((1, vocab + 1), dtype=BF16, device="cuda"), torch.zeros((1, 1), device="cuda"), 4)
