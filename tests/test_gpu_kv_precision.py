"""GPU: attention results against 64 bits, as close as 32-bit sums and 24-bit
operands make them (tests/kv_ref.py: result_bound), in every shape of the
kernel: a cluster a unit, equal shares, one and two tiles of queries."""

from __future__ import annotations

import pytest
import torch
from kv_ref import attend_exact, result_bound, result_error

from expertrelay_b200 import kv

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _even_cache(gen, rows, kv_heads, n, d, ps, dtype):
    """Rows of n positions in pages of ps; n is a multiple of ps. Returns the cache and k, v [rows, kv_heads, n, d]."""
    each = n // ps
    k, v = (torch.randn((rows * each, kv_heads, ps, d), generator=gen, device="cuda").to(dtype) for _ in range(2))
    table = torch.randperm(rows * each, generator=gen, device="cuda").to(torch.int32).view(rows, each)
    seen = [x[table.long()].transpose(1, 2).reshape(rows, kv_heads, n, d) for x in (k, v)]
    return kv.PagedKV(k, v, table), *seen


@pytest.mark.parametrize(("cache_dtype", "q_dtype"), [(BF16, BF16), (BF16, F32), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize(("rows", "kv_heads", "group", "n", "d"), [
    (64, 4, 4, 1008, 64), (64, 4, 4, 1008, 128), (32, 2, 8, 1008, 256), (32, 2, 16, 1008, 64), (32, 2, 16, 1008, 128),
    (32, 2, 12, 1008, 256), (64, 4, 2, 48, 64), (64, 4, 2, 144, 32), (4, 2, 16, 32000, 64), (4, 4, 8, 32000, 128),
    (1, 2, 8, 480, 128), (2, 1, 16, 2000, 64), (24, 2, 7, 2000, 96), (16, 2, 8, 4000, 192),
])
@pytest.mark.parametrize("size", [1.0, 0.02])
def test_attend_is_as_exact_as_32_bits(cuda, cache_dtype, q_dtype, rows, kv_heads, group, n, d, size):
    """size: the spread of the scores. Near zero they are exact enough that the weights and their sums alone count."""
    gen = torch.Generator(device="cuda").manual_seed(n + d)
    cache, k, v = _even_cache(gen, rows, kv_heads, n, d, 16, cache_dtype)
    lens = torch.full((rows,), n, dtype=torch.int32, device="cuda")
    # bf16 results show few of their errors: new queries until there are results enough
    calls = 1 if q_dtype == F32 else max(1, 400000 // (rows * kv_heads * group * d))
    outs, wants = [], []
    for _ in range(calls):
        q = torch.randn((rows, kv_heads * group, d), generator=gen, device="cuda").to(q_dtype)
        outs.append(kv.attend(cache, q, lens, scale=size * d ** -0.5))
        wants.append(attend_exact(q.view(rows, kv_heads, group, d), k, v, size * d ** -0.5))
    got = result_error(torch.stack(outs), torch.stack(wants), q_dtype)
    assert got <= result_bound(d, n, size), f"{got:.3g} of the result, {result_bound(d, n, size):.3g} allowed"
    cache.check()
