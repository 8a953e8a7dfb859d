"""What the precision tests of attention see (tests/kv_ref.py: result_bound, result_error): arithmetic that loses a
part of an operand is outside the bound, at every head size and length; arithmetic in 32 bits, and with the
products that the kernels leave out, is inside it."""

from __future__ import annotations

import pytest
import torch
from kv_ref import attend_exact, result_bound, result_error

F32, BF16 = torch.float32, torch.bfloat16


def _cut(x, bits):
    """The leading `bits` bits of fp32 values, as float64."""
    return (x.view(torch.int32) & -(1 << (24 - bits))).view(F32).double()


def _parts(x, n, last_rounded=True):
    """The sum of the first n bf16 parts of fp32 values, cut, the last one rounded."""
    total, rest = torch.zeros_like(x, dtype=torch.float64), x.clone()
    for i in range(n):
        part = rest.to(BF16).double() if i == n - 1 and last_rounded else _cut(rest, 8)
        total += part
        rest = (x.double() - total).float()
    return total


def _attend(q, k, v, scale, weight=lambda p: p.double(), left_out=None):
    """In 64 bits from the operands given, the weights by `weight`; left_out(a, b) is taken off each product sum."""
    s = torch.einsum("rhgd,rhnd->rhgn", q.double(), k.double())
    if left_out:
        s = s - torch.einsum("rhgd,rhnd->rhgn", *(x.double() for x in left_out(q, k)))
    p = torch.exp((s - s.amax(-1, keepdim=True)) * scale).float()
    out = torch.einsum("rhgn,rhnd->rhgd", weight(p), v.double())
    if left_out:
        out = out - torch.einsum("rhgn,rhnd->rhgd", *(x.double() for x in left_out(p, v)))
    return out / p.double().sum(-1, keepdim=True)


def _inputs(d, n, rows, cache):
    gen = torch.Generator().manual_seed(d + n)
    q = torch.randn((rows, 1, 8, d), generator=gen)
    k, v = (torch.randn((rows, 1, n, d), generator=gen).to(cache).float() for _ in range(2))
    return q, k, v


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [20, 333, 1501, 32000])
@pytest.mark.parametrize("size", [1.0, 0.02])
def test_lost_parts_are_seen_in_fp32_results(d, n, size):
    scale, bound = size * d ** -0.5, result_bound(d, n, size)
    lead = lambda x: _cut(x, 11)  # noqa: E731
    # the rests of 11-bit operands, the two of which the fp32-cache kernel does not multiply
    rests = lambda a, b: (a - lead(a).float(), b - lead(b).float())  # noqa: E731
    q, k, v = _inputs(d, n, 2, F32)
    want = attend_exact(q, k, v, scale)
    err = lambda got: result_error(got.float(), want, F32)  # noqa: E731
    p = torch.softmax(torch.einsum("rhgd,rhnd->rhgn", q, k) * scale, -1)
    assert err(torch.einsum("rhgn,rhnd->rhgd", p, v)) <= bound  # 32 bits throughout
    assert err(_attend(q, k, v, scale)) <= bound
    assert err(_attend(q, k, v, scale, left_out=rests)) <= bound
    assert err(_attend(q, k, lead(v), scale)) > 3 * bound
    assert err(_attend(q, k, v, scale, weight=lead)) > 3 * bound
    if size == 1.0:  # scores near zero hide what is lost of their operands
        assert err(_attend(lead(q), k, v, scale)) > 3 * bound
        assert err(_attend(q, lead(k), v, scale)) > 3 * bound
    q, k, v = _inputs(d, n, 2, BF16)
    want = attend_exact(q, k, v, scale)
    assert err(_attend(_parts(q, 3), k, v, scale, weight=lambda p: _parts(p, 3))) <= bound
    if size == 1.0:
        assert err(_attend(_parts(q, 2, last_rounded=False), k, v, scale)) > 1.5 * bound
    elif n <= 1501:  # over 32000 keys the bound has room for the running sums' rounding
        assert err(_attend(q, k, v, scale, weight=lambda p: _parts(p, 2))) > 1.5 * bound


@pytest.mark.parametrize(("d", "n"), [(64, 48), (128, 333), (256, 1008)])
def test_lost_parts_are_seen_in_bf16_results(d, n):
    size = 0.02
    scale, bound = size * d ** -0.5, result_bound(d, n, size)
    q, k, v = _inputs(d, n, 400000 // (8 * d), BF16)
    q = q.to(BF16).float()
    want = attend_exact(q, k, v, scale)
    err = lambda got: result_error(got.to(BF16), want, BF16)  # noqa: E731
    p = torch.softmax(torch.einsum("rhgd,rhnd->rhgn", q, k) * scale, -1)
    assert err(torch.einsum("rhgn,rhnd->rhgd", p, v)) <= bound
    assert err(_attend(q, k, v, scale, weight=lambda p: _parts(p, 3))) <= bound
    assert err(_attend(q, k, v, scale, weight=lambda p: _parts(p, 2))) > 2 * bound
    assert err(_attend(q, k, v, scale, weight=lambda p: _parts(p, 1))) > 30 * bound
