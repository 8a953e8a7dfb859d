"""Trees of drafted tokens, copies of pages and beam selection by their definitions, for the tests."""

from __future__ import annotations

import math

import numpy as np
from kv_ref import attend_row, attend_tolerance, tokens


def paths(parents):
    """Each node's ancestors and itself, ascending."""
    got = []
    for i, p in enumerate(parents):
        got.append((got[p] if p >= 0 else []) + [i])
    return got


def check_trees(cache, q, lens, trees, out, *, first=0, seqs=None, scale=None, skip=()):
    """trees: the parents of each one. Every node's row of `out` against 64 bits (kv_ref's tolerance)."""
    d = cache.head_dim
    scale = d ** -0.5 if scale is None else scale
    table = cache.table.cpu()
    at = first
    for t, parents in enumerate(trees):
        n, m = lens[t], len(parents)
        s = t if seqs is None else seqs[t]
        kk, vv = tokens(cache.k, table, s, n + m), tokens(cache.v, table, s, n + m)
        for i, path in enumerate(paths(parents)):
            if t not in skip:
                see = np.array(list(range(n)) + [n + j for j in path])
                want, _, spread, size = attend_row(q[at].double().cpu().numpy(), kk[:, see], vv[:, see], scale)
                tol = attend_tolerance(want, spread, size, d, len(see), out.dtype)
                got = out[at].double().cpu().numpy()
                assert np.all(np.abs(got - want) <= tol), (f"tree {t}, node {i} of {m} after {n}: off by "
                                                           f"{np.max(np.abs(got - want) / tol):.3g} of the tolerance")
            at += 1


def beam_reference(logits, scores, count):
    """logits [batch, beams, vocab], scores [batch, beams] float64 numpy -> per batch the best (value, beam, token)."""
    result = []
    for rows, score in zip(logits, scores):
        pairs = []
        for b, row in enumerate(rows):
            top = row.max()
            fine = not np.isnan(row).any() and np.isfinite(top) and np.isfinite(score[b])
            lse = top + math.log(np.exp(row - top).sum()) if fine else 0.0
            value = np.where(np.isneginf(row) | (not fine), -np.inf, score[b] + (row - lse))
            pairs += [(-v, b * len(row) + i) for i, v in enumerate(value)]
        pairs = sorted(pairs)[:count]
        result.append([(-v, at // rows.shape[1], at % rows.shape[1]) for v, at in pairs])
    return result
