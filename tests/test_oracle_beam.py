"""The beam-search oracle against what its definition says on problems small enough to enumerate."""

import itertools
import math

import numpy as np

from oracle import beam


def log_softmax(x):
    x = np.asarray(x, np.float64)
    return x - math.log(np.exp(x).sum())


def test_candidates_by_enumeration():
    g = np.random.default_rng(0)
    rows, scores = g.normal(size=(3, 7)), g.normal(size=3).astype(np.float32)
    want = sorted(((-(float(scores[b]) + log_softmax(rows[b])[i]), b, i)
                   for b in range(3) for i in range(7)))
    got = beam.group_candidates(list(rows), scores, 21)
    assert [(b, i) for _, b, i in got] == [(b, i) for _, b, i in want]
    assert np.allclose([t for t, _, _ in got], [-t for t, _, _ in want])
    assert beam.group_candidates(list(rows), scores, 4) == got[:4]


def test_ties_go_to_the_lower_beam_then_token():
    rows = [np.zeros(4), np.zeros(4)]
    got = beam.group_candidates(rows, np.zeros(2, np.float32), 6)
    assert [(b, i) for _, b, i in got] == [(0, 0), (0, 1), (0, 2), (0, 3), (1, 0), (1, 1)]


def test_rows_that_propose_nothing():
    ok = np.array([0.0, -np.inf, 1.0])
    rows = [np.full(3, -np.inf), np.array([0.0, np.nan, 1.0]), np.array([0.0, np.inf, 1.0]), ok, ok]
    got = beam.group_candidates(rows, np.array([0, 0, 0, -np.inf, -1], np.float32), 9)
    assert [(b, i) for _, b, i in got] == [(4, 2), (4, 0)]


def new_state(G, W, T):
    s = {"scores": np.full((G, W), -np.inf, np.float32), "lengths": np.zeros(G, np.int32),
         "done": np.zeros(G, bool), "finished_scores": np.full((G, W), -np.inf, np.float32),
         "finished_beams": np.full((G, W), -1), "finished_token_ids": np.full((G, W), -1),
         "finished_lengths": np.zeros((G, W), int), "token_history": np.full((G, T, W), -1),
         "parent_history": np.full((G, T, W), -1)}
    s["scores"][:, 0] = 0
    return s


def test_a_wide_search_finds_the_best_sequences():
    """As many beams as prefixes: beam search is exhaustive.  The model's rows depend on the last
    token only; token 0 stops."""
    V, T, W, alpha = 3, 3, 12, 0.7
    table = np.random.default_rng(5).normal(size=(V, V))
    prompt = np.random.default_rng(6).normal(size=V)
    s = new_state(1, W, T)
    for t in range(T):
        last = s["token_history"][0, t - 1] if t else np.full(W, -1)
        s = beam.step(lambda g, w: table[last[w]] if t else prompt, s, [0], alpha)
        s = {k: v for k, v in s.items() if k not in ("token_ids", "parents")}
    ids, lengths, scores = beam.finish(s, W, alpha)
    every = []
    for n in range(1, T + 1):
        for seq in itertools.product(range(V), repeat=n):
            if 0 in seq[:-1] or (seq[-1] != 0 and n < T):
                continue
            rows = [prompt] + [table[c] for c in seq[:-1]]
            total = sum(log_softmax(r)[c] for r, c in zip(rows, seq))
            every.append((-total / n ** alpha, seq))
    every.sort()
    best = [seq for _, seq in every[:5]]
    # done may end the search once W hypotheses are finished, never before the best five here
    assert [tuple(ids[0, j, :lengths[0, j]]) for j in range(5)] == best
    assert np.allclose(scores[0, :5], [-v for v, _ in every[:5]])


def test_stop_tokens_below_rank_w_end_nothing():
    s = new_state(1, 2, 4)
    s["scores"][0] = [0.0, -0.1]
    rows = [np.array([2.0, 5.0, 1.0, -9.0]), np.array([2.0, 5.0, 1.0, -9.0])]
    got = beam.step(lambda g, w: rows[w], s, [0], 1.0)
    # ranks 0 and 1 are (0, 1), (1, 1); the stop token 0 has rank 2 and 3
    assert got["token_ids"].tolist() == [[1, 1]] and got["parents"].tolist() == [[0, 1]]
    assert np.isneginf(got["finished_scores"]).all() and not got["done"][0]
    got = beam.step(lambda g, w: rows[w], s, [1], 1.0)
    # both of rank below 2 stop; the next two of the six candidates go on
    assert got["finished_token_ids"].tolist() == [[1, 1]]
    assert got["finished_beams"].tolist() == [[0, 1]]
    assert got["token_ids"].tolist() == [[0, 0]] and got["parents"].tolist() == [[0, 1]]
    assert bool(got["done"][0])  # two finished, and both better than what runs


def test_finish_follows_the_parents():
    s = new_state(1, 2, 3)
    s["lengths"][:] = 3
    s["token_history"][0] = [[10, 11], [20, 21], [30, 31]]
    s["parent_history"][0] = [[0, 0], [1, 0], [1, 0]]
    s["scores"][0] = [-3.0, -6.0]
    ids, lengths, scores = beam.finish(s, 2, 1.0)
    assert ids.tolist() == [[[10, 21, 30], [11, 20, 31]]]
    assert lengths.tolist() == [[3, 3]] and scores.tolist() == [[-1.0, -2.0]]


def test_reorder_reads_the_rows_before_the_call():
    x = np.arange(6 * 4).reshape(6, 4)
    got = beam.reorder(x, np.array([[1, 0, 1], [-1, 7, 0]]), lengths=np.array([2, 4]))
    want = x.copy()
    want[0, :2], want[1, :2], want[2, :2] = x[1, :2], x[0, :2], x[1, :2]
    want[5] = x[3]
    assert (got == want).all()


def test_a_running_beam_without_a_recorded_parent_is_its_own():
    s = new_state(1, 3, 4)
    s["token_history"] = np.arange(12).reshape(1, 4, 3)
    s["parent_history"] = np.array([[[0, 1, 2], [0, 1, 2], [-1, 7, 0], [0, 0, 0]]])
    s["scores"] = np.array([[-1.0, -2.0, -3.0]], np.float32)
    s["lengths"][0] = 3
    ids, lengths, _ = beam.finish(s, 3)
    assert lengths.tolist() == [[3, 3, 3]]
    assert ids[0, :, :3].tolist() == [[0, 3, 6], [1, 4, 7], [0, 3, 8]]
