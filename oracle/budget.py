"""Packed prompt attention, the attention weight keys receive, and caches held at a budget, in 64 bits (oracle).

Definitions, one sequence of ``nq`` queries and ``nk`` keys at a time: ``x_ij = scale q_i . k_j``, with a soft cap
``c tanh(x / c)``; query ``i`` sees the keys ``j <= i + nk - nq``; ``lse_i = log(sum_j exp(x_ij) + exp(sink))``;
``o_i = sum_j exp(x_ij - lse_i) v_j`` over the keys it sees only. The mass of key ``j`` is the sum of ``exp(x_ij - lse_i)``
over the queries that see it and the query heads of its KV head.

Pinned by (``tests/test_oracle_budget.py``): loops over single pairs, the masses' sum (a weight of one per query and head),
and a selection by sorting tuples.
"""

from __future__ import annotations

import numpy as np

__all__ = ["attention_mass", "evict", "heavy_step", "prompt_attention"]


def _scores(q, k, scale, softcap):
    x = scale * (q @ k.T)
    return softcap * np.tanh(x / softcap) if softcap else x


def _seen(nq, nk):
    return np.arange(nk)[None, :] <= np.arange(nq)[:, None] + nk - nq


def _bounds(rows):
    if isinstance(rows, tuple):
        return list(zip(*(np.asarray(r).tolist() for r in rows)))
    rows = np.asarray(rows).tolist()
    return list(zip(rows[:-1], rows[1:]))


def prompt_attention(q, k, v, rows_q, rows_k, scale, softcap=None, sinks=None):
    """``q [T, Hq, D]``, ``k`` / ``v`` ``[Tk, Hkv, D]``: out ``[T, Hq, D]``, lse ``[Hq, T]`` and ``sum_j p_ij |v_j|``
    ``[T, Hq, D]`` (what a relative error of the weights can change), all float64."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    heads, groups = q.shape[1], q.shape[1] // k.shape[1]
    out, size = np.zeros(q.shape), np.zeros(q.shape)
    lse = np.full((heads, q.shape[0]), -np.inf)
    for (q0, q1), (k0, k1) in zip(_bounds(rows_q), _bounds(rows_k)):
        seen = _seen(q1 - q0, k1 - k0)
        for h in range(heads):
            with np.errstate(invalid="ignore", over="ignore"):
                x = _scores(q[q0:q1, h], k[k0:k1, h // groups], scale, softcap)
            for i in range(q1 - q0):  # over the keys it sees only: the others may hold anything
                xi = x[i][seen[i]]
                vi = v[k0:k1, h // groups][seen[i]]
                full = xi if sinks is None else np.append(xi, float(sinks[h]))
                if not len(full):
                    continue
                m = full.max()
                lse[h, q0 + i] = m + np.log(np.exp(full - m).sum())
                p = np.exp(xi - lse[h, q0 + i])
                with np.errstate(invalid="ignore"):
                    out[q0 + i, h] = p @ vi
                    size[q0 + i, h] = p @ np.abs(vi)
    return out, lse, size


def attention_mass(q, k, lse, rows_q, rows_k, scale, softcap=None, window=None):
    """``[Hkv, Tk]`` float64."""
    q, k, lse = (np.asarray(x, np.float64) for x in (q, k, lse))
    heads, groups = q.shape[1], q.shape[1] // k.shape[1]
    mass = np.zeros((k.shape[1], k.shape[0]))
    for (q0, q1), (k0, k1) in zip(_bounds(rows_q), _bounds(rows_k)):
        seen = _seen(q1 - q0, k1 - k0)
        if window:
            seen[: max(0, q1 - q0 - window)] = False
        for h in range(heads):
            with np.errstate(invalid="ignore", over="ignore"):
                x = _scores(q[q0:q1, h], k[k0:k1, h // groups], scale, softcap)
                p = np.where(seen, np.exp(np.where(seen, x, 0.0) - np.where(seen, lse[h, q0:q1, None], 0.0)), 0.0)
            mass[h // groups, k0:k1] += p.sum(0)
    return mass


def _order(score):
    """What scores are compared by: a NaN is the least."""
    return np.where(np.isnan(score), -np.inf, score)


def evict(mass, budget, recent, first):
    """The tokens of one row and head that stay, ascending: ``mass [n]``."""
    n = len(mass)
    if n <= budget:
        return np.arange(n)
    must = [j for j in range(n) if j < first or j >= n - recent]
    # (a NaN is less than minus infinity: it sorts by a second key)
    others = sorted((j for j in range(n) if first <= j < n - recent),
                    key=lambda j: (bool(np.isnan(mass[j])), -_order(mass)[j], j))
    return np.array(sorted(must + others[: budget - len(must)]), np.int64)


def heavy_step(state, q, k, v, budget, recent, first, scale, softcap=None, sinks=None):
    """One row's step, in place on ``state`` (keys / values ``[Hkv, C, D]``, score, position ``[Hkv, C]`` float64 / int,
    count ``[Hkv]``, length int): ``q [Hq, D]``, ``k`` / ``v`` ``[Hkv, D]``; out ``[Hq, D]`` and ``sum_j p_j |v_j|``."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    kv_heads = k.shape[0]
    groups = q.shape[0] // kv_heads
    out, size = np.zeros(q.shape), np.zeros(q.shape)
    t = state["length"]
    for h in range(kv_heads):
        n = state["count"][h]
        if n < budget:
            to, n = n, n + 1
        else:
            pos, score = state["position"][h], state["score"][h]
            free = [s for s in range(budget) if first <= pos[s] <= t - recent]
            to = min(free, key=lambda s: (not np.isnan(score[s]), _order(score)[s], s)) if free else 0
        state["keys"][h, to], state["values"][h, to] = k[h], v[h]
        state["score"][h, to], state["position"][h, to] = 0.0, t
        state["count"][h] = n
        for g in range(groups):
            head = h * groups + g
            x = _scores(q[head][None], state["keys"][h, :n], scale, softcap)[0]
            full = x if sinks is None else np.append(x, float(sinks[head]))
            m = full.max()
            p = np.exp(x - m) / np.exp(full - m).sum()
            out[head] = p @ state["values"][h, :n]
            size[head] = p @ np.abs(state["values"][h, :n])
            state["score"][h, :n] += p
    state["length"] = t + 1
    return out, size
