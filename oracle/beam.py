"""CPU restatement of beam search in 64 bits (numpy), one group at a time.

Test infrastructure only: nothing in the product path imports it.  The operators are defined in
include/mvsd.h (beam_select, beam_step, beam_reorder, beam_finish); the reference has none."""

from __future__ import annotations

import numpy as np

NINF = -np.inf


def row_logsum(x: np.ndarray) -> float:
    """log sum exp of a row in 64 bits; not finite for a row of -inf or one with a NaN or +inf."""
    x = np.asarray(x, np.float64)
    top = x.max() if x.size else NINF
    if not np.isfinite(top):  # NaN propagates through max
        return float("nan")
    return float(top + np.log(np.exp(x - top).sum()))


def group_candidates(rows: list, scores: np.ndarray, count: int) -> list:
    """[(total, beam, token)] of one group, best first: rows[b] is beam b's row."""
    found = []
    for b, row in enumerate(rows):
        s = float(np.float32(scores[b]))
        if not np.isfinite(s):
            continue
        x = np.asarray(row, np.float64)
        lse = row_logsum(x)
        if not np.isfinite(lse):
            continue
        order = np.lexsort((np.arange(x.size), -x))[:count]
        found += [(-(s + (x[i] - lse)), b, -x[i], int(i)) for i in order if x[i] > NINF]
    found.sort()
    return [(-t, b, i) for t, b, _, i in found[:count]]


def select(rows_of, scores: np.ndarray, count: int):
    """token ids, parents, scores [G, count]; rows_of(g, w) gives a row."""
    G, W = scores.shape
    ids, parents = np.full((G, count), -1), np.full((G, count), -1)
    out = np.full((G, count), NINF)
    for g in range(G):
        got = group_candidates([rows_of(g, w) for w in range(W)], scores[g], count)
        for j, (t, b, i) in enumerate(got):
            ids[g, j], parents[g, j], out[g, j] = i, b, t
    return ids, parents, out


def step(rows_of, state: dict, stops=(), length_penalty=1.0, early_stopping=False) -> dict:
    """The state after a step (arrays as in BeamState) with its token_ids and parents."""
    new = {k: np.array(v, copy=True) for k, v in state.items()}
    new["scores"] = new["scores"].astype(np.float64)
    new["finished_scores"] = new["finished_scores"].astype(np.float64)
    G, T, W = state["token_history"].shape
    new["token_ids"], new["parents"] = np.full((G, W), -1), np.full((G, W), -1)
    stops = {int(s) for s in stops}
    for g in range(G):
        length = int(state["lengths"][g])
        if state["done"][g] or not 0 <= length < T:
            continue
        got = group_candidates([rows_of(g, w) for w in range(W)], state["scores"][g],
                               W * (1 + len(stops)))
        power = float(length + 1) ** length_penalty
        pool = [tuple(new["finished_" + k][g, j] for k in ("scores", "beams", "token_ids",
                                                           "lengths"))
                for j in range(W) if state["finished_scores"][g, j] > NINF]
        pool += [(t / power, b, i, length + 1) for t, b, i in got[:W] if i in stops]
        pool.sort(key=lambda h: -h[0])
        pool = pool[:W]
        going = [c for c in got if c[2] not in stops][:W]
        over = not going or (len(pool) == W and (early_stopping
                                                 or pool[-1][0] >= going[0][0] / power))
        going += [(NINF, -1, -1)] * (W - len(going))
        new["done"][g], new["lengths"][g] = over, length + 1
        new["scores"][g] = [t for t, _, _ in going]
        new["parents"][g] = new["parent_history"][g, length] = [b for _, b, _ in going]
        new["token_ids"][g] = new["token_history"][g, length] = [i for _, _, i in going]
        pool += [(NINF, -1, -1, 0)] * (W - len(pool))
        for j, k in enumerate(("scores", "beams", "token_ids", "lengths")):
            new["finished_" + k][g] = [h[j] for h in pool]
    return new


def finish(state: dict, count: int, length_penalty=1.0):
    """token ids [G, count, T], lengths and scores [G, count]."""
    G, T, W = state["token_history"].shape
    ids = np.full((G, count, T), -1)
    lengths, scores = np.zeros((G, count), np.int64), np.full((G, count), NINF)
    for g in range(G):
        pool = [tuple(state["finished_" + k][g, j] for k in ("scores", "beams", "token_ids",
                                                             "lengths"))
                for j in range(W) if state["finished_scores"][g, j] > NINF]
        at = min(max(int(state["lengths"][g]), 0), T)
        if not state["done"][g] and at > 0:
            parents = [int(p) if 0 <= p < W else w
                       for w, p in enumerate(state["parent_history"][g, at - 1])]
            pool += [(float(s) / float(at) ** length_penalty, parents[w],
                      state["token_history"][g, at - 1, w], at)
                     for w, s in enumerate(state["scores"][g]) if np.isfinite(s)]
        pool.sort(key=lambda h: -h[0])
        for j, (s, b, t, n) in enumerate(pool[:count]):
            n = min(max(int(n), 0), T)
            scores[g, j], lengths[g, j] = s, n
            if n < 1:
                continue
            b = int(b) if 0 <= b < W else 0
            ids[g, j, n - 1] = t
            for k in range(n - 2, -1, -1):
                ids[g, j, k] = state["token_history"][g, k, b]
                parent = int(state["parent_history"][g, k, b])
                b = parent if 0 <= parent < W else b
    return ids, lengths, scores


def reorder(x: np.ndarray, parents: np.ndarray, starts=None, lengths=None, length_dim=1,
            slots=None, out=None) -> np.ndarray:
    """The reordered states (a copy of x, or of out with its rows written)."""
    G, W = parents.shape
    new = np.array(x if out is None else out, copy=True)
    T = x.shape[length_dim]
    for g in range(G):
        a = 0 if starts is None else min(max(int(starts[g]), 0), T)
        b = T if lengths is None else min(int(lengths[g]), T)
        if b <= a:
            continue
        at = (slice(None),) * (length_dim - 1) + (slice(a, b),)
        for w in range(W):
            p = int(parents[g, w])
            p = p if 0 <= p < W else w
            src, dst = (g * W + p, g * W + w) if slots is None else (slots[g, p], slots[g, w])
            if 0 <= src < x.shape[0] and 0 <= dst < x.shape[0]:
                new[dst][at] = x[src][at]
    return new
