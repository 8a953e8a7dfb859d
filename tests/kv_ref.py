"""The paged cache's operators in 64 bits, row by row, and seeded caches for the tests."""

from __future__ import annotations

import numpy as np
import torch

STEP = np.float32(1) / np.float32(127)  # a code's step, relative to the greatest magnitude
U = 2.0 ** -23  # one truncating 32-bit addition (a rounded one is off by half of it)


def half_step(dtype) -> float:
    """The most one rounding to `dtype` is off, relative to the value."""
    return torch.finfo(dtype).eps / 2


def make_cache(gen, lens, kv_heads, d, ps, dtype, *, layout="hnd", spare=2, width=None, device="cuda"):
    """Pools with the sequences' pages strewn over them and NaN in every slot no
    sequence uses; layout "hnd" ([page, head, slot, d]), "nhd" (stored
    [page, slot, head, d]) or "wide" (every slot in a wider row)."""
    counts = [-(-n // ps) for n in lens]
    pages = sum(counts) + spare
    w = max([1, *counts]) if width is None else width
    stored = {"hnd": (pages, kv_heads, ps, d), "nhd": (pages, ps, kv_heads, d), "wide": (pages, kv_heads, ps, d + 8)}[layout]
    k, v = (torch.full(stored, float("nan"), dtype=dtype, device=device) for _ in range(2))
    k, v = ((x.transpose(1, 2) if layout == "nhd" else x[..., :d]) for x in (k, v))
    table = torch.full((len(lens), w), -1, dtype=torch.int32)
    order = torch.randperm(pages, generator=gen)
    at = 0
    for s, n in enumerate(lens):
        table[s, : counts[s]] = order[at:at + counts[s]].to(torch.int32)
        at += counts[s]
        kk, vv = (torch.randn((kv_heads, n, d), generator=gen).to(dtype).to(device) for _ in range(2))
        for i in range(counts[s]):
            m = min(ps, n - i * ps)
            k[int(table[s, i]), :, :m] = kk[:, i * ps:i * ps + m]
            v[int(table[s, i]), :, :m] = vv[:, i * ps:i * ps + m]
    return k, v, table.to(device)


def tokens(pool, table, s, n):
    """[kv_heads, n, d] float64: sequence s's first n positions."""
    ps = pool.shape[2]
    out = np.zeros((pool.shape[1], n, pool.shape[3]))
    for i in range(-(-n // ps)):
        m = min(ps, n - i * ps)
        out[:, i * ps:i * ps + m] = pool[int(table[s, i]), :, :m].double().cpu().numpy()
    return out


def attend_row(q, k, v, scale, pick=None):
    """q [heads, d], k, v [kv_heads, n, d] -> out [heads, d], weights
    [kv_heads, n], and for each output the bound factors: sum p |v| and the
    greatest sum |q k| scale."""
    heads, d = q.shape
    kv_heads, n, _ = k.shape
    group = heads // kv_heads
    out, spread, mass, size = np.zeros((heads, d)), np.zeros((heads, d)), np.zeros((kv_heads, n)), 0.0
    for h in range(heads):
        kh = h // group
        at = np.arange(n) if pick is None else pick[kh]
        if len(at) == 0:
            continue
        s = (k[kh, at] @ q[h]) * scale
        if np.all(s == -np.inf):
            continue
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h] = p @ v[kh, at]
        spread[h] = p @ np.abs(v[kh, at])
        mass[kh, at] += p
        size = max(size, float((np.abs(k[kh, at]) @ np.abs(q[h])).max() * scale))
    return out, mass, spread, size


def attend_tolerance(out, spread, size, d, n, dtype):
    """What the kernels may be off. A score is d products and sums in 32 bits,
    then a scale and a subtraction: off by (d + 4) U size. That moves a weight
    and the sum below by its exponential, so 2 (d + 4) U size relative to
    sum p |v|; the weights (rounded to 16 + 8 bits on the tensor cores: 2^-16),
    their sum and the sum over n positions add 2^-16 + (2 n + 16) U; then one
    rounding of the result."""
    eps = 2 * (d + 4) * U * size + 2.0 ** -16 + (2 * n + 16) * U
    return eps * spread + half_step(dtype) * np.abs(out) + 1e-30


def bounds_of(keys):
    """keys [n, d] float32 numpy -> (lo codes, hi codes, scale)."""
    lo, hi = keys.min(0), keys.max(0)
    scale = np.float32(max(np.abs(lo).max(), np.abs(hi).max()) * STEP)
    if scale == 0:
        return np.zeros_like(lo, dtype=np.int8), np.zeros_like(hi, dtype=np.int8), scale
    return np.rint(lo / scale).astype(np.int8), np.rint(hi / scale).astype(np.int8), scale


def choose(score, n, budget, first, last):
    """Ordinals kept of n by score, as the selections define it."""
    if n <= budget:
        return list(range(n))
    mid = list(range(first, n - last))
    rank = sorted(mid, key=lambda i: (-(score[i]) if not np.isnan(score[i]) else np.inf, i))
    # NaN after -inf: they compare equal in the key above, so put them last by hand
    rank = [i for i in rank if not np.isnan(score[i])] + [i for i in rank if np.isnan(score[i])]
    return sorted(list(range(first)) + rank[: budget - first - last] + list(range(n - last, n)))


def page_scores(q, codes_lo, codes_hi, scales):
    """q [group, d] float32, codes [n, d] int8, scales [n] float32 -> [n] float32."""
    with np.errstate(invalid="ignore", divide="ignore"):
        t = (np.abs(q).max(1) * STEP).astype(np.float32)
        c = np.rint(q / np.where(t == 0, np.float32(1), t)[:, None]).astype(np.float32)
        c = np.nan_to_num(c, nan=0.0).astype(np.int64)
        whole = np.maximum(c, 0) @ codes_hi.T.astype(np.int64) + np.minimum(c, 0) @ codes_lo.T.astype(np.int64)
        return ((whole.astype(np.float32) * t[:, None]).max(0) * scales).astype(np.float32)


def result_bound(d, n, size=1.0):
    """The most an attention result may be off before its own rounding, as a
    share (2-norm) of the result, with 32-bit sums and 24-bit operands over
    normal inputs. size: the spread of the scores (1 where scale is d^-0.5).

    A score is at most d / 8 matrix products added up one after another, each
    cutting the sum by up to U of what it is so far. The sum grows as the square
    root, so the cuts come to no more than half of U (d / 8) of the score, and
    change its weight by that times the score: (d / 16) size U. The operands'
    last bits, the product of their rests where that is left out (2^-21 at the
    most, 2^-23.6 on average), exponentials, weights and the two sums over a
    chunk of keys: 4 U together. Running sums over n / 16 chunks are rounded:
    half of U each at the most, a third of that on average, of a sum that
    grows as the square root too: sqrt(n / 16) U / 4 covers it."""
    return (d / 16 * size + 4 + (n / 16) ** 0.5 / 4) * U


def result_error(out, want, dtype):
    """How far `out` (tensor of dtype, one row's results or many of one size)
    is from the 64-bit `want` before its rounding, as a share of the 2-norm.
    In 32 bits that is what is seen. A bf16 result shows an error only where
    it crosses the border between two bf16 values: with chance |error| / step,
    and then by a step. So the squares of (out - rounded want) add up to the sum of
    |error| step, and |error| is 0.8 of its root mean square for normal ones."""
    out, want = out.double().flatten(), want.double().flatten()
    rms = want.pow(2).mean().sqrt()
    if dtype == torch.float32:
        return float((out - want).pow(2).mean().sqrt() / rms)
    right = want.to(dtype).double()
    step = torch.exp2(torch.floor(torch.log2(right.abs().clamp(min=1e-30))) - 7)
    return float((out - right).pow(2).sum() / (0.8 * rms * step.sum()))


def attend_exact(q, k, v, scale):
    """q [rows, kv_heads, group, d], k, v [rows, kv_heads, n, d] -> results, in 64 bits."""
    p = torch.softmax(torch.einsum("rhgd,rhnd->rhgn", q.double(), k.double()) * scale, -1)
    return torch.einsum("rhgn,rhnd->rhgd", p, v.double())
