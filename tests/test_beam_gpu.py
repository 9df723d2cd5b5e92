"""Beam search on the device against the 64-bit oracle (oracle/beam.py).

Token ids, parents, lengths and flags are exact.  Scores: a total is formed in 64 bits from the
row's lse and rounded once (2^-24 relative).  The lse carries the error of its fp32 sums: a term's
exponent is the rounded product of a rounded difference, 2.2 * 2^-24 relative, at most 40 in
magnitude where the term counts, times ln 2; v_exp_f32 is good to 2^-23; a lane adds up to 32 terms,
then ten more additions.  (2.2 * 40 * 0.7 + 2 + 42) * 2^-24 = 6.3e-6 at most."""

import math

import numpy as np
import pytest
import torch

from mvsd.sample import (BeamSearch, BeamState, beam_search_finish, beam_search_select,
                         beam_search_step, reorder_beams)
from oracle import beam as oracle

pytestmark = pytest.mark.gpu

LSE_ERROR = 6.3e-6
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def close(got, want, scale=1.0):
    got, want = got.double().cpu().numpy(), np.asarray(want, np.float64)
    fine = np.isfinite(want)
    assert np.array_equal(fine, np.isfinite(got))
    assert np.array_equal(got[~fine], want[~fine])
    bar = LSE_ERROR * scale + 2.0 ** -22 * np.abs(want[fine])
    assert (np.abs(got[fine] - want[fine]) <= bar).all()


def rows_of(x, W, rows=None):
    host = x.double().cpu().numpy()
    return lambda g, w: host[g * W + w if rows is None else int(rows[g, w])]


def make_scores(device, G, W, seed, alive=None):
    s = -20 - np.cumsum(np.random.default_rng(seed).exponential(0.4, (G, W)), axis=1)
    if alive is not None:
        s[:, alive:] = -np.inf
    return torch.tensor(s, dtype=torch.float32, device=device)


def check_select(x, scores, C, rows=None):
    got = beam_search_select(x, scores, C, target_rows=rows)
    W = scores.shape[1]
    ids, parents, want = oracle.select(rows_of(x, W, rows), scores.cpu().numpy(), C)
    assert np.array_equal(got.token_ids.cpu().numpy(), ids)
    assert np.array_equal(got.parents.cpu().numpy(), parents)
    close(got.scores, want)
    return got


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [1, 3, 7, 9, 63, 500, 2047, 2049, 8191, 8193, 50257])
@pytest.mark.parametrize("G,W,C", [(1, 1, 1), (2, 4, 8), (1, 5, 256), (3, 17, 40)])
def test_select_edges(device, dtype, V, G, W, C):
    gen = torch.Generator(device=device).manual_seed(V * 7 + W)
    x = (torch.randn(G * W, V, device=device, generator=gen) * 2.5).to(DTYPES[dtype])
    check_select(x, make_scores(device, G, W, V), C)
    if V > 2:  # a view: rows start at an odd element and are not adjacent
        check_select(x[:, 1:], make_scores(device, G, W, V), C)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("alive", [1, 3, 8])
def test_select_long_chunks(device, dtype, alive):
    """Enough rows for the long chunks, a full vocabulary, beams that do not run."""
    G, W, V = 16, 8, 151936
    gen = torch.Generator(device=device).manual_seed(alive)
    x = (torch.randn(G * W, V, device=device, generator=gen) * 2.5).to(DTYPES[dtype])
    scores = make_scores(device, G, W, alive, alive)
    x[alive:W] = math.nan  # rows of absent beams are not looked at
    check_select(x, scores, 16)


def test_select_64_beams(device):
    G, W, V = 2, 64, 3001
    x = torch.randn(G * W, V, device=device, generator=torch.Generator(device=device).manual_seed(0))
    check_select(x, make_scores(device, G, W, 1), 256)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_select_masked_rows(device, dtype):
    """Rows of -inf, of the type's lowest value, with NaN or infinities; whole groups of them."""
    G, W, V, C = 6, 4, 9000, 8
    t = DTYPES[dtype]
    low = torch.finfo(t).min
    gen = torch.Generator(device=device).manual_seed(3)
    x = (torch.randn(G * W, V, device=device, generator=gen) * 2).to(t)
    x[0] = -math.inf
    x[1, :8999] = -math.inf          # one token allowed
    x[2, 17] = math.nan
    x[3, 8998] = math.inf
    x[4:8] = -math.inf               # a group that cannot go on
    x[8:12, 5:] = -math.inf          # five tokens a beam
    x[12:16] = low                   # masked by the lowest value, one token allowed
    x[12:16, 77] = 1.0
    x[16] = low                      # nothing but the lowest value
    x[17:20] = 0.0                   # uniform rows
    x[20:24] = x[20:24].float().round().to(t)  # long runs of equal values
    got = check_select(x, make_scores(device, G, W, 2), C)
    assert (got.parents[1] == -1).all()
    check_select(x, make_scores(device, G, W, 4), 33)
    scores = make_scores(device, G, W, 2)
    scores[0, 0], scores[2, 1], scores[3, 2] = math.nan, math.inf, -math.inf
    check_select(x, scores, C)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [4000, 151936])
@pytest.mark.parametrize("C", [8, 256])
def test_select_runs_of_equal_values(device, dtype, V, C):
    """More entries at the bound than the gather holds: the lowest beams and tokens win."""
    G, W = 2, 4
    x = torch.zeros(G * W, V, device=device, dtype=DTYPES[dtype])
    x[5, V // 2:] = 3.0
    x[6, V - 3] = 9.0
    scores = torch.zeros(G, W, device=device)
    scores[1] = torch.tensor([-1.0, -1.0, -0.5, 0.0], device=device)
    check_select(x, scores, C)
    x[:] = torch.finfo(x.dtype).min
    check_select(x, scores, C)
    x[:, ::2] = -math.inf
    check_select(x, scores, C)


def test_negative_zero_ties_with_zero(device):
    x = torch.full((2, 700), -5.0, device=device)
    x[0, [3, 600]] = torch.tensor([-0.0, 0.0], device=device)
    x[1, [2, 5, 9]] = torch.tensor([0.0, -0.0, 0.0], device=device)
    got = check_select(x, torch.zeros(1, 2, device=device), 5)
    assert got.token_ids.tolist() == [[3, 600, 2, 5, 9]] or \
        got.token_ids.tolist() == [[2, 5, 9, 3, 600]]


def test_select_reads_rows_by_index(device):
    G, W, V = 3, 4, 4099
    gen = torch.Generator(device=device).manual_seed(9)
    big = torch.randn(40, V + 5, device=device, generator=gen).to(torch.bfloat16)[:, 3:3 + V]
    rows = torch.randperm(40, device=device, generator=gen)[:G * W].view(G, W).to(torch.int32)
    scores = make_scores(device, G, W, 0)
    check_select(big, scores, 8, rows)
    # indices outside the tensor read its nearest row
    out = rows.clone()
    out[0, 0], out[1, 1], out[2, 2] = -5, 40, 2 ** 31 - 1
    inside = out.clamp(0, 39)
    a, b = (beam_search_select(big, scores, 8, target_rows=r) for r in (out, inside))
    assert torch.equal(a.token_ids, b.token_ids) and torch.equal(a.scores, b.scores)
    # the same row for every beam: beams differ by their scores only
    check_select(big, scores, 8, torch.zeros_like(rows))
    check_select(big[:1].expand(G * W, V), scores, 8)


def test_order_of_two_beams_is_that_of_the_64_bit_totals(device):
    """Totals of two beams one fp32 rounding apart keep their order."""
    V = 5000
    row = torch.randn(V, device=device, generator=torch.Generator(device=device).manual_seed(4))
    x = row.repeat(2, 1)
    for ulps in (1, 2, 40):
        s = torch.tensor([[-20.0, -20.0]], device=device)
        s[0, 1] += ulps * 2.0 ** -19  # an ulp of 20 is 2^-19
        got = check_select(x, s, 6)
        assert got.parents[0].tolist() == [1, 0, 1, 0, 1, 0]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("V", [700, 9001, 50257])
@pytest.mark.parametrize("heavier", [0, 1])
def test_near_ties_follow_the_64_bit_totals(device, dtype, V, heavier):
    """Two beams with the same logits in opposite orders, so that fp32 sums differ, and one of them
    with a little more mass: its totals are lower by about 1e-8, far below what fp32 sums resolve and
    far above what 64-bit ones do."""
    G = 48
    gen = torch.Generator(device=device).manual_seed(V)
    x = (torch.randn(G, 2, V, device=device, generator=gen) * 2.5).to(DTYPES[dtype])
    x[:, 0, V // 2] = x[:, 0, V - 1 - V // 2] = -math.inf  # the places that the flip maps there
    x[:, 1] = x[:, 0].flip(-1)
    lse = torch.logsumexp(x[:, heavier].double(), dim=-1)
    x[:, heavier, V // 2] = (lse + math.log(1e-8)).to(x.dtype)
    scores = torch.full((G, 2), -20.0, device=device)
    got = check_select(x.reshape(2 * G, V), scores, 6)
    assert (got.parents[:, 0] == 1 - heavier).all()
    # at the last place: the better of the two is in, the other one is not
    got = check_select(x.reshape(2 * G, V), scores, 1)
    assert (got.parents[:, 0] == 1 - heavier).all()


@pytest.mark.parametrize("heavier", [0, 1])
def test_near_ties_of_totals_around_zero(device, heavier):
    """Scores that bring the best totals to zero, where a bound in proportion to them is none."""
    G, V = 64, 9001
    gen = torch.Generator(device=device).manual_seed(heavier)
    x = torch.randn(G, 2, V, device=device, generator=gen) * 2.5
    x[:, 0, V // 2] = -math.inf
    x[:, 1] = x[:, 0].flip(-1)
    lse = torch.logsumexp(x[:, heavier].double(), dim=-1)
    x[:, heavier, V // 2] = (lse + math.log(1e-8)).float()
    scores = (lse - x[:, 0].amax(-1).double()).float()[:, None].expand(G, 2).contiguous()
    for C in (1, 2, 3):
        got = check_select(x.reshape(2 * G, V), scores, C)
        assert (got.parents[:, 0] == 1 - heavier).all()


@pytest.mark.parametrize("dtype,last", [("fp32", 7171), ("bf16", 6151)])
@pytest.mark.parametrize("G", [2, 512])
@pytest.mark.parametrize("heavier", [0, 1])
def test_near_ties_of_rows_with_one_large_entry(device, dtype, last, G, heavier):
    """An entry beside which each of the others vanishes in fp32 (5.6e-8 of it), but not their sum:
    first or last in the order of columns.  (512 groups: rows long enough for the long chunks.)"""
    V = 8192
    x = torch.full((G, 2, V), -16.7, device=device, dtype=DTYPES[dtype])
    x[:, 0, 0] = x[:, 1, last] = 0.0
    x[:, :, 5000] = -math.inf
    x[:, heavier, 5000] = math.log(1e-8)
    got = check_select(x.reshape(2 * G, V), torch.full((G, 2), -20.0, device=device), 2)
    assert (got.parents == torch.tensor([1 - heavier, heavier], device=device)).all()


def test_equal_beams_in_front_of_large_masks(device):
    """Masked tokens at -1e9: totals that 64 bits hold to 1e-7, of beams with the same mass."""
    G, V = 48, 30000
    gen = torch.Generator(device=device).manual_seed(2)
    x = torch.full((G, 2, V), -1e9, device=device)
    x[:, 0, 100:141] = torch.randn(G, 41, device=device, generator=gen)
    x[:, 1] = x[:, 0].flip(-1)
    check_select(x.reshape(2 * G, V), torch.full((G, 2), -20.0, device=device), 100)


@pytest.mark.parametrize("large", [1e10, -1e10, 1e30, -1e30])
def test_near_ties_of_huge_logits(device, large):
    """Logits so large that nothing but their maximum counts: two of it in one beam, three in the
    others, of which two are equal."""
    x = torch.full((3, 9001), -abs(large) * 4, device=device)
    x[:, 5] = x[:, 8000] = x[1:, 40] = large
    check_select(x, torch.full((1, 3), -20.0, device=device), 8)


@pytest.mark.parametrize("heavier", [0, 1])
def test_near_ties_in_front_of_masked_tokens(device, heavier):
    """Two tokens a beam allowed, the others at the type's lowest value: the last places are runs of
    that value, the first ones near ties of the two beams (mass 1e-8 apart)."""
    V = 30000
    x = torch.full((2, V), torch.finfo(torch.float32).min, device=device)
    x[:, 100], x[:, 20000] = 1.0, 0.25
    lse = math.log(math.exp(1.0) + math.exp(0.25))
    x[heavier, 7] = lse + math.log(1e-8)
    scores = torch.tensor([[-20.0, -20.0]], device=device)
    got = check_select(x, scores, 12)
    assert got.parents[0, :2].tolist() == [1 - heavier, heavier]
    assert got.token_ids[0, :4].tolist() == [100, 100, 20000, 20000]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("C", [8, 40, 256])
def test_rows_in_order(device, dtype, C):
    """The largest entries side by side (more above the bound than the gather holds)."""
    G, W, V = 2, 3, 60001
    gen = torch.Generator(device=device).manual_seed(C)
    x = (torch.randn(G * W, V, device=device, generator=gen) * 2.5).to(DTYPES[dtype])
    x[:3] = x[:3].sort(dim=-1, descending=True).values
    x[4] = x[4].sort(dim=-1).values
    check_select(x, make_scores(device, G, W, 1), C)


def test_huge_offsets(device):
    """Rows whose element offsets pass 2^31 (bf16, a row stride of 2^29)."""
    V, stride = 1500, 2 ** 29
    base = torch.zeros(5 * stride + V, device=device, dtype=torch.bfloat16)
    x = base.as_strided((6, V), (stride, 1))
    x.copy_(torch.randn(6, V, device=device, generator=torch.Generator(device=device).manual_seed(8)))
    check_select(x, make_scores(device, 2, 3, 5), 6)


def test_threads_on_one_stream(device):
    """Two threads enqueue on the same stream, selections and steps of different sizes."""
    import threading

    gen = torch.Generator(device=device).manual_seed(3)
    work = []
    for G, W, V in ((3, 4, 30011), (2, 8, 9001)):
        x = torch.randn(G * W, V, device=device, generator=gen) * 2.5
        scores = make_scores(device, G, W, V)
        work.append((x, scores, beam_search_select(x, scores, 16)))
    torch.cuda.synchronize(device)
    wrong = []

    def run(x, scores, want):
        for _ in range(200):
            got = beam_search_select(x, scores, 16)
            if not torch.equal(got.token_ids, want.token_ids):
                wrong.append(1)

    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_empty_batch(device):
    got = beam_search_select(torch.zeros(0, 10, device=device), torch.zeros(0, 4, device=device), 8)
    assert got.token_ids.shape == (0, 8)
    state = BeamState.new(0, 4, 8, device)
    assert beam_search_step(torch.zeros(0, 10, device=device), state).parents.shape == (0, 4)
    assert beam_search_finish(state).token_ids.shape == (0, 4, 8)
    assert reorder_beams([], torch.zeros(2, 4, dtype=torch.int32, device=device)) == []


# ----------------------------------------------------------------- step


def host(state):
    return {k: v.cpu().numpy() for k, v in vars(state).items()}


def random_state(device, G, W, T, seed, done=(), full=()):
    r = np.random.default_rng(seed)
    s = BeamState.new(G, W, T, device)
    s.scores = make_scores(device, G, W, seed)
    lengths = r.integers(0, T, G)
    lengths[list(full)] = T
    s.lengths = torch.tensor(lengths, dtype=torch.int32, device=device)
    s.done[list(done)] = True
    fs = -np.sort(r.exponential(2.0, (G, W)), axis=1)
    none = np.arange(W)[None] >= r.integers(0, W + 1, G)[:, None]
    fs[none] = -np.inf
    fb, ft, fl = r.integers(0, W, (G, W)), r.integers(0, 99, (G, W)), r.integers(1, T + 1, (G, W))
    fb[none], ft[none], fl[none] = -1, -1, 0

    def put(v, dtype=torch.int32):
        return torch.tensor(v, dtype=dtype, device=device)

    s.finished_scores = put(fs, torch.float32)
    s.finished_beams, s.finished_token_ids, s.finished_lengths = put(fb), put(ft), put(fl)
    s.token_history = put(r.integers(0, 99, (G, T, W)))
    s.parent_history = put(r.integers(0, W, (G, T, W)))
    return s


def clone(state):
    return BeamState(**{k: v.clone() for k, v in vars(state).items()})


def check_state(got, want):
    for k, v in vars(got).items():
        if k.endswith("scores"):
            close(v, want[k])
        else:
            assert np.array_equal(v.cpu().numpy(), want[k]), k


def check_step(x, state, stops, alpha=1.0, early=False, rows=None):
    want = oracle.step(rows_of(x, state.scores.shape[1], rows), host(state), stops, alpha, early)
    ids = torch.tensor(stops, dtype=torch.int32, device=x.device)
    out = clone(state)  # separate arrays for the new state, the histories shared
    mine = clone(state)
    out.token_history, out.parent_history = mine.token_history, mine.parent_history
    before = {k: v.clone() for k, v in vars(mine).items() if not k.endswith("history")}
    got = beam_search_step(x, mine, stop_token_ids=ids, length_penalty=alpha,
                           early_stopping=early, target_rows=rows, out=out)
    check_state(got.state, want)
    assert np.array_equal(got.token_ids.cpu().numpy(), want["token_ids"])
    assert np.array_equal(got.parents.cpu().numpy(), want["parents"])
    for k, v in before.items():  # the old state is left as it was
        assert torch.equal(getattr(mine, k), v), k
    # and in place
    inside = clone(state)
    here = beam_search_step(x, inside, stop_token_ids=ids, length_penalty=alpha,
                            early_stopping=early, target_rows=rows)
    assert here.state is inside
    for k, v in vars(out).items():
        assert torch.equal(v, getattr(inside, k)), k
    assert torch.equal(here.token_ids, got.token_ids)
    return got, want


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("G,W,V,E", [(1, 1, 50, 1), (9, 4, 700, 2), (5, 8, 2100, 0), (3, 12, 9001, 5),
                                     (2, 64, 4100, 3), (1, 128 // 2, 40, 1)])
@pytest.mark.parametrize("alpha,early", [(1.0, False), (0.0, True), (0.6, False)])
def test_step(device, dtype, G, W, V, E, alpha, early):
    gen = torch.Generator(device=device).manual_seed(G * 100 + W)
    x = (torch.randn(G * W, V, device=device, generator=gen) * 2.5).to(DTYPES[dtype])
    stops = np.random.default_rng(W).permutation(V)[:E].tolist()
    if E:  # a third of the rows want to stop
        want = torch.rand(G * W, 1, device=device, generator=gen) < 0.33
        at = torch.tensor(stops, device=device)
        x[:, at] = torch.where(want, torch.full_like(x[:, at], 9.0), x[:, at])
    state = random_state(device, G, W, 20, W, done=[1] if G > 2 else [], full=[2] if G > 2 else [])
    check_step(x, state, stops, alpha, early)


def test_step_groups_that_rest(device):
    """Done and full groups, lengths outside the histories, a group whose rows are masked."""
    G, W, V, T = 6, 3, 600, 5
    x = torch.randn(G * W, V, device=device, generator=torch.Generator(device=device).manual_seed(1))
    state = random_state(device, G, W, T, 3, done=[0], full=[1])
    state.lengths[2] = -4
    state.lengths[3] = 2 ** 31 - 1
    x[4 * W:5 * W] = -math.inf
    state.done[4] = state.done[5] = False
    state.lengths[4:] = 2
    got, _ = check_step(x, state, [7])
    assert got.token_ids[:5].eq(-1).all() and got.state.done[4] and not got.state.done[5]
    # resting groups' rows are not looked at
    y = x.clone()
    y[:4 * W] = math.nan
    again = beam_search_step(y, clone(state), stop_token_ids=torch.tensor([7], dtype=torch.int32,
                                                                          device=device))
    assert torch.equal(again.token_ids, got.token_ids)


def test_step_all_candidates_stop(device):
    """Only stop tokens are allowed: nothing runs on, the group is done."""
    W, V = 4, 300
    x = torch.full((W, V), -math.inf, device=device)
    x[:, 5], x[:, 9] = 1.0, 0.5
    state = BeamState.new(1, W, 6, device)
    state.scores = make_scores(device, 1, W, 0)
    got, want = check_step(x, state, [9, 5])
    assert bool(got.state.done[0]) and torch.isneginf(got.state.scores).all()
    assert want["finished_scores"][0, 0] > -np.inf


def test_equal_hypotheses_keep_the_earlier_one(device):
    W, V = 2, 64
    x = torch.zeros(W, V, device=device)
    state = BeamState.new(1, W, 8, device)
    lp = -math.log(64.0)
    state.scores = torch.tensor([[0.0, 0.0]], device=device)
    state.finished_scores = torch.tensor([[lp, lp]], dtype=torch.float32, device=device)
    state.finished_beams = torch.tensor([[1, 0]], dtype=torch.int32, device=device)
    state.finished_token_ids = torch.tensor([[40, 41]], dtype=torch.int32, device=device)
    state.finished_lengths = torch.tensor([[1, 1]], dtype=torch.int32, device=device)
    # a sum of 64 ones is exact, and so is what follows from it in 64 bits
    stop = torch.tensor([0, 1], dtype=torch.int32, device=device)
    got = beam_search_step(x, state, stop_token_ids=stop)
    assert got.state.finished_token_ids.tolist() == [[40, 41]]
    assert bool(got.state.done[0]) and got.token_ids.tolist() == [[2, 3]]
    assert got.parents.tolist() == [[0, 0]]


# ----------------------------------------------------------------- reorder


def values(device, shape, dtype, seed):
    gen = torch.Generator(device=device).manual_seed(seed)
    if dtype.is_floating_point:
        return torch.randn(shape, device=device, generator=gen).to(dtype)
    most = 2 if dtype == torch.bool else 200
    return torch.randint(0, most, shape, device=device, generator=gen).to(dtype)


def as_bytes(x):
    return x.contiguous().view(torch.uint8).cpu().numpy().reshape(x.shape + (-1,))


def check_reorder(x, parents, length_dim=1, **kw):
    """In place and out of place against the oracle, byte for byte."""
    args = {k: None if v is None else v.cpu().numpy() for k, v in kw.items()}
    raw = as_bytes(x)
    want = oracle.reorder(raw, parents.cpu().numpy(), length_dim=length_dim, **args)
    out = values(x.device, x.shape, x.dtype, 77)
    want_out = oracle.reorder(raw, parents.cpu().numpy(), length_dim=length_dim, out=as_bytes(out),
                              **args)
    assert reorder_beams(x, parents, length_dim=length_dim, out=out, **kw) is out
    assert np.array_equal(as_bytes(out), want_out)
    assert np.array_equal(as_bytes(x), raw)  # the states are left alone
    assert reorder_beams(x, parents, length_dim=length_dim, **kw) is x
    assert np.array_equal(as_bytes(x), want)


def make_parents(device, G, W, seed):
    r = np.random.default_rng(seed)
    p = r.integers(0, W, (G, W))
    p[0] = np.roll(np.arange(W), 1)  # a cycle through every row
    if G > 1:
        p[1] = W - 1                 # one heir of all
    if G > 2:
        p[2] = -1                    # a group that rests
    if G > 3:
        p[3, 0], p[3, -1] = W, 2 ** 31 - 1  # outside: kept
    return torch.tensor(p, dtype=torch.int32, device=device)


def counts(device, G, T, seed):
    n = np.random.default_rng(seed).integers(0, T + 1, G)
    n[0] = T
    if G > 1:
        n[1] = 1
    if G > 4:
        n[3], n[4] = 0, T + 100      # nothing; past the end: the tensor's length
    return torch.tensor(n, dtype=torch.int32, device=device)


@pytest.mark.parametrize("W", [1, 2, 5, 8, 9, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("shape,dim,dtype", [
    ((37,), 1, torch.int32), ((1,), 1, torch.int64), ((3, 19, 5), 2, torch.float16),
    ((70, 2, 3), 1, torch.bfloat16), ((2, 3, 13, 1), 3, torch.uint8), ((259,), 1, torch.bool),
    ((33, 16), 1, torch.float32)])
def test_reorder(device, W, shape, dim, dtype):
    G = 6
    x = values(device, (G * W, *shape), dtype, W)
    T = shape[dim - 1]
    check_reorder(x, make_parents(device, G, W, W), dim)
    check_reorder(x, make_parents(device, G, W, W), dim, lengths=counts(device, G, T, W))
    starts = torch.tensor([0, 1, T // 2, T + 5, -3, T // 3], dtype=torch.int32, device=device)
    check_reorder(x, make_parents(device, G, W, 2 * W), dim, starts=starts)
    check_reorder(x, make_parents(device, G, W, 3 * W), dim, starts=starts,
                  lengths=counts(device, G, T, 2 * W))


@pytest.mark.parametrize("W", [2, 4, 20])
def test_reorder_pages_through_slots(device, W):
    """The last pages of the beams in a pool; slots outside it are left alone, and so is the rest."""
    G, pages = 5, 300
    x = values(device, (pages, 16, 3, 8), torch.bfloat16, W)
    order = np.random.default_rng(W).permutation(pages)[:G * W].reshape(G, W)
    slots = torch.tensor(order, dtype=torch.int32, device=device)
    slots[0, 0], slots[1, 1] = -1, pages
    check_reorder(x, make_parents(device, G, W, 1), 1, slots=slots,
                  lengths=counts(device, G, 16, 3))


def test_reorder_views(device):
    """Rows apart from each other, off a vector's alignment, keys and values in one tensor."""
    G, W = 3, 4
    parents = make_parents(device, G, W, 5)
    base = values(device, (G * W, 2, 9, 7), torch.float16, 0)
    want = np.stack([oracle.reorder(as_bytes(base[:, k]), parents.cpu().numpy())
                     for k in range(2)], axis=1)
    reorder_beams([base[:, 0], base[:, 1]], parents)
    assert np.array_equal(as_bytes(base), want)
    wide = values(device, (G * W, 50), torch.uint8, 1)
    keep = wide.clone()
    part = wide[:, 3:44]
    want = oracle.reorder(as_bytes(part), parents.cpu().numpy())
    reorder_beams(part, parents)
    assert np.array_equal(as_bytes(part), want)
    assert torch.equal(wide[:, :3], keep[:, :3]) and torch.equal(wide[:, 44:], keep[:, 44:])
    # more rows than beams: those behind the last are left as they were
    more = values(device, (G * W + 3, 20), torch.int32, 2)
    tail = more[G * W:].clone()
    reorder_beams(more, parents)
    assert torch.equal(more[G * W:], tail)


def test_reorder_takes_an_iterator(device):
    parents = torch.tensor([[1, 0]], dtype=torch.int32, device=device)
    states = [values(device, (2, 5), torch.int32, k) for k in range(3)]
    want = [x.flip(0) for x in states]
    got = reorder_beams(iter(states), parents)
    assert all(torch.equal(x, w) for x, w in zip(got, want)) and len(got) == 3


def test_reorder_many_tensors(device):
    """More states than one launch takes, of different shapes and types, empty ones among them."""
    G, W = 4, 3
    parents = make_parents(device, G, W, 2)
    shapes = [(G * W, 11), (G * W, 0), (G * W, 40, 2), (G * W, 11, 0), (G * W + 5, 200)]
    states = [values(device, shapes[k % 5], [torch.int32, torch.bfloat16][k % 2], k)
              for k in range(60)]
    want = [oracle.reorder(as_bytes(x), parents.cpu().numpy()) if x.numel() else None
            for x in states]
    got = reorder_beams(states, parents)
    for x, y, w in zip(states, got, want):
        assert y is x
        if w is not None:
            assert np.array_equal(as_bytes(x), w)


def test_reorder_states_of_one_call_once(device):
    """Empty states among many, through the C ABI: none is reordered twice."""
    import ctypes

    from mvsd import _native as nat

    parents = torch.tensor([[1, 2, 0]], dtype=torch.int32, device=device)
    states = [values(device, (3, 9), torch.uint8, k) for k in range(60)]
    want = [x[[1, 2, 0]] for x in states]
    flat = []
    for k, x in enumerate(states):
        flat += [x.data_ptr(), x.data_ptr(), 9, 9, 3, 1, 9, 1]
        if k % 3 == 0:
            flat += [x.data_ptr(), x.data_ptr(), 9, 9, 3, 1, 0, 1]  # no entries
    assert nat.lib().mvsd_beam_reorder((ctypes.c_int64 * len(flat))(*flat), len(flat) // 8,
                                       parents.data_ptr(), None, None, None, 1, 3,
                                       nat.stream_of(device)) == 0
    assert all(torch.equal(x, w) for x, w in zip(states, want))


def test_reorder_many_groups(device):
    """More (group, state) pairs than one grid has rows."""
    G, W = 3000, 2
    r = np.random.default_rng(0)
    parents = torch.tensor(r.integers(0, W, (G, W)), dtype=torch.int32, device=device)
    states = [values(device, (G * W, 5), torch.int32, k) for k in range(24)]
    src = (torch.arange(G, device=device)[:, None] * W + parents).view(-1).long()
    want = [x[src] for x in states]
    reorder_beams(states, parents)
    assert all(torch.equal(x, w) for x, w in zip(states, want))


def test_reorder_huge_offsets(device):
    """Rows beyond 4 GiB."""
    W, T, D = 3, 1_000_000, 800
    x = torch.empty((2 * W, T, D), dtype=torch.uint8, device=device)
    for r in range(2 * W):
        x[r] = r + 1
    parents = torch.tensor([[1, 2, 0], [0, 0, 1]], dtype=torch.int32, device=device)
    n = torch.tensor([T, 999_999], dtype=torch.int32, device=device)
    reorder_beams(x, parents, lengths=n)
    assert [int(x[r, T - 2, D - 1]) for r in range(6)] == [2, 3, 1, 4, 4, 5]
    assert [int(x[r, T - 1, 0]) for r in range(6)] == [2, 3, 1, 4, 5, 6]
    assert [int(x[r, 0, 0]) for r in range(6)] == [2, 3, 1, 4, 4, 5]


def test_reorder_refusals(device):
    x = torch.zeros(8, 10, device=device)
    parents = torch.zeros(2, 4, dtype=torch.int32, device=device)
    for bad in (dict(out=x[:, :].view(8, 10)), dict(out=torch.zeros(8, 11, device=device)),
                dict(out=[x, x]), dict(length_dim=2), dict(length_dim=0),
                dict(lengths=torch.zeros(3, dtype=torch.int32, device=device)),
                dict(slots=torch.zeros(8, dtype=torch.int32, device=device)),
                dict(lengths=torch.zeros(2, dtype=torch.int32))):
        if "out" in bad and isinstance(bad["out"], torch.Tensor) and bad["out"].shape == x.shape:
            assert reorder_beams(x, parents, **bad) is bad["out"]  # the same memory: in place
            continue
        with pytest.raises((ValueError, NotImplementedError)):
            reorder_beams(x, parents, **bad)
    with pytest.raises(TypeError):
        reorder_beams(x, parents.long())
    with pytest.raises(ValueError):
        reorder_beams(x[:7], parents)
    with pytest.raises(ValueError):
        reorder_beams(x.t(), torch.zeros(1, 4, dtype=torch.int32, device=device))
    with pytest.raises(ValueError, match="share memory"):
        reorder_beams([x, x], parents)
    with pytest.raises(ValueError, match="share memory"):
        reorder_beams(x[:4], parents[:1], out=x[2:6])
    with pytest.raises(ValueError):
        reorder_beams(x.expand(2, 8, 10).transpose(0, 1), parents)


# ----------------------------------------------------------------- finish


@pytest.mark.parametrize("G,W,T,n", [(1, 1, 1, 1), (1, 4, 2, 4), (7, 3, 33, 2), (5, 8, 300, 8),
                                     (2, 64, 130, 64), (3, 5, 4097, 1), (1, 2, 20000, 2)])
@pytest.mark.parametrize("alpha", [0.0, 1.0])
def test_finish(device, G, W, T, n, alpha):
    state = random_state(device, G, W, T, T + W, done=[1] if G > 2 else [],
                         full=[0])
    before = {k: v.clone() for k, v in vars(state).items()}
    got = beam_search_finish(state, n, length_penalty=alpha)
    ids, lengths, scores = oracle.finish(host(state), n, alpha)
    assert np.array_equal(got.token_ids.cpu().numpy(), ids)
    assert np.array_equal(got.lengths.cpu().numpy(), lengths)
    close(got.scores, scores)
    for k, v in before.items():
        assert torch.equal(getattr(state, k), v)


def test_finish_of_odd_histories(device):
    """Parents outside the group, lengths outside the histories, beams that are none."""
    G, W, T = 4, 3, 50
    state = random_state(device, G, W, T, 11)
    r = np.random.default_rng(1)
    state.parent_history = torch.tensor(r.integers(-2, W + 3, (G, T, W)), dtype=torch.int32,
                                        device=device)
    state.lengths = torch.tensor([0, -7, 2 ** 31 - 1, 9], dtype=torch.int32, device=device)
    state.finished_lengths[0, 0] = 2 ** 31 - 1
    state.finished_scores[0, 0], state.finished_beams[0, 0] = -0.5, 99
    state.scores[3] = torch.tensor([-1.0, math.nan, -math.inf], device=device)
    got = beam_search_finish(state)
    ids, lengths, scores = oracle.finish(host(state), W, 1.0)
    assert np.array_equal(got.token_ids.cpu().numpy(), ids)
    assert np.array_equal(got.lengths.cpu().numpy(), lengths)
    close(got.scores, scores)


# ----------------------------------------------------------------- together


class Chain:
    """A tiny model with a state: the next row depends on the sum of the beam's cached tokens."""

    def __init__(self, device, V, seed):
        gen = torch.Generator(device=device).manual_seed(seed)
        self.V, self.table = V, torch.randn(V, V, device=device, generator=gen) * 2

    def rows(self, cache, length):
        return self.table[(cache[:, :length].sum(dim=1) % self.V)]


@pytest.mark.parametrize("G,W,alpha,early", [(1, 4, 1.0, False), (5, 3, 0.6, True)])
def test_a_whole_search(device, G, W, alpha, early):
    """step, reorder and finish together, as a server runs them, against the oracle's own search."""
    V, T = 23, 12
    model = Chain(device, V, 0)
    table = model.table.double().cpu().numpy()
    search = BeamSearch(G, W, T, device, stop_token_ids=[0, 4], length_penalty=alpha,
                        early_stopping=early)
    cache = torch.zeros(G * W, T + 1, dtype=torch.int64, device=device)
    cache[:, 0] = torch.arange(G, device=device).repeat_interleave(W) * 5 + 1
    mine = {k: v.copy() for k, v in host(search.state).items()}
    prefix = [[[g * 5 + 1]] * W for g in range(G)]
    for t in range(T):
        step = search.step(model.rows(cache, t + 1))
        search.reorder(cache, lengths=torch.full((G,), t + 1, dtype=torch.int32, device=device))
        cache[:, t + 1] = step.token_ids.view(-1).clamp(min=0)
        want = oracle.step(lambda g, w: table[sum(prefix[g][w]) % V], mine, [0, 4], alpha, early)
        assert np.array_equal(step.token_ids.cpu().numpy(), want["token_ids"])
        assert np.array_equal(step.parents.cpu().numpy(), want["parents"])
        prefix = [[prefix[g][max(want["parents"][g, w], 0)] + [max(int(want["token_ids"][g, w]), 0)]
                   if want["parents"][g, w] >= 0 else prefix[g][w] + [0]
                   for w in range(W)] for g in range(G)]
        mine = {k: want[k] for k in mine}
    got = search.finish()
    ids, lengths, scores = oracle.finish(mine, W, alpha)
    assert np.array_equal(got.token_ids.cpu().numpy(), ids)
    assert np.array_equal(got.lengths.cpu().numpy(), lengths)
    close(got.scores, scores, scale=T)


def test_streams_and_graphs(device):
    """Two captured steps, replayed several times and beside eager work, share no scratch."""
    G, W, V, T = 3, 4, 5003, 6
    gen = torch.Generator(device=device).manual_seed(0)
    rows = [torch.randn(G * W, V, device=device, generator=gen) for _ in range(2)]
    states = [random_state(device, G, W, T, k) for k in range(2)]
    for s in states:
        s.lengths.fill_(2)
        s.done.fill_(False)
    caches = [values(device, (G * W, 77), torch.int32, k) for k in range(2)]
    stop = torch.tensor([3], dtype=torch.int32, device=device)

    def work(k, state, cache, out):
        step = beam_search_step(rows[k], state, stop_token_ids=stop, out=out)
        return step, reorder_beams(cache, step.parents, out=torch.zeros_like(cache)), \
            beam_search_finish(out)

    def separate(state):
        out = clone(state)
        out.token_history, out.parent_history = state.token_history, state.parent_history
        return out

    want = []
    for k in range(2):
        s = clone(states[k])
        want.append(work(k, s, caches[k], separate(s)))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graphs, got, inputs = [], [], []
    for k in range(2):
        s = clone(states[k])
        o = separate(s)
        inputs.append(s)  # a graph reads its inputs' memory at every replay
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            work(k, s, caches[k], o)  # warm
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(work(k, s, caches[k], o))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for graph, stream in zip(graphs, streams):  # both in flight
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
        beam_search_select(rows[0], states[0].scores, 8)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a[0].token_ids, b[0].token_ids)
            assert torch.equal(a[0].parents, b[0].parents)
            assert torch.equal(a[0].state.scores, b[0].state.scores)
            assert torch.equal(a[1], b[1])
            assert torch.equal(a[2].token_ids, b[2].token_ids)


def test_scratch_grows_and_is_kept_per_stream(device):
    """Calls of growing and shrinking sizes on two streams at once."""
    sizes = [(1, 4, 500), (8, 8, 30000), (2, 3, 9000), (64, 8, 50257), (1, 1, 40), (64, 8, 50257)]
    cases = []
    for k, (G, W, V) in enumerate(sizes):
        gen = torch.Generator(device=device).manual_seed(k)
        cases.append((torch.randn(G * W, V, device=device, generator=gen), make_scores(device, G, W, k)))
    want = [beam_search_select(x, s, 8) for x, s in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for x, s in cases * 3:
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[k].append(beam_search_select(x, s, 8))
    torch.cuda.synchronize()
    for mine in got:
        for a, b in zip(mine, want * 3):
            assert torch.equal(a.token_ids, b.token_ids) and torch.equal(a.scores, b.scores)


def test_same_results_twice(device):
    G, W, V = 16, 8, 32000
    gen = torch.Generator(device=device).manual_seed(0)
    x = (torch.randn(G * W, V, device=device, generator=gen) * 2).to(torch.bfloat16)
    s = make_scores(device, G, W, 0)
    a = [beam_search_select(x, s, 16) for _ in range(4)]
    for b in a[1:]:
        assert torch.equal(a[0].scores, b.scores) and torch.equal(a[0].token_ids, b.token_ids)


def test_refusals(device):
    x = torch.zeros(8, 100, device=device)
    s = torch.zeros(2, 4, device=device)
    i32 = dict(dtype=torch.int32, device=device)
    for bad in (lambda: beam_search_select(x, s, 0), lambda: beam_search_select(x, s, 257),
                lambda: beam_search_select(x[:7], s, 8), lambda: beam_search_select(x.t(), s[:1], 8),
                lambda: beam_search_select(x, s[0], 8), lambda: beam_search_select(x, s[:, ::2], 4),
                lambda: beam_search_select(x, torch.zeros(1, 65, device=device), 4),
                lambda: beam_search_select(x, torch.zeros(1, 0, device=device), 4),
                lambda: beam_search_select(x[:, :0], s, 4),
                lambda: beam_search_select(x, s, 8, target_rows=torch.zeros(3, **i32)),
                lambda: beam_search_finish(BeamState.new(2, 4, 8, device), 5),
                lambda: beam_search_finish(BeamState.new(2, 4, 8, device), 0),
                lambda: beam_search_step(x, BeamState.new(2, 4, 8, device),
                                         stop_token_ids=torch.zeros(64, **i32)),
                lambda: beam_search_step(x, BeamState.new(2, 4, 8, device),
                                         out=BeamState.new(2, 4, 8, device)),
                lambda: beam_search_step(x[:7], BeamState.new(2, 4, 8, device)),
                lambda: beam_search_step(x, BeamState.new(2, 4, 8, device),
                                         length_penalty=math.nan),
                lambda: beam_search_finish(BeamState.new(2, 4, 8, device),
                                           length_penalty=math.inf)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: beam_search_select(x.double(), s, 8),
                lambda: beam_search_select(x, s.double(), 8),
                lambda: beam_search_select(x, s, 8, target_rows=torch.zeros(2, 4, dtype=torch.int64,
                                                                            device=device))):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(NotImplementedError):
        beam_search_select(x, s.cpu(), 8)


# ----------------------------------------------------------------- rows shorter than a vector


def short_rows(device, dtype, V, G=4):
    """Groups of four beams: +inf in the first one's row, a NaN in the second's, +inf throughout a row
    whose beam has no finite score, and a fourth beam that goes on (in the last group not even that)."""
    gen = torch.Generator(device=device).manual_seed(V)
    x = torch.randn(G * 4, V, device=device, generator=gen).to(DTYPES[dtype])
    x[0::4, V // 2] = math.inf
    x[1::4, V - 1] = math.nan
    x[2::4] = math.inf
    x[-1] = math.inf
    scores = make_scores(device, G, 4, V)
    for g in range(G):
        scores[g, 2] = (-math.inf, math.nan, math.inf, -math.inf)[g % 4]
    return x, scores


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [1, 2, 3, 4, 5, 7, 8, 9])
def test_short_rows_of_beams_that_propose_nothing(device, dtype, V):
    x, scores = short_rows(device, dtype, V)
    for C in (1, V, 40, 256):
        got = check_select(x, scores, C)
        assert (got.parents[:-1, :min(C, V)] == 3).all() and (got.parents[-1] == -1).all()
    state = random_state(device, 4, 4, 9, V)
    state.scores = scores
    # (not check_step, which compares the old state with itself: one of its scores is a NaN)
    want = oracle.step(rows_of(x, 4), host(state), [0, 2])
    got = beam_search_step(x, state, stop_token_ids=torch.tensor([0, 2], dtype=torch.int32,
                                                                 device=device))
    check_state(got.state, want)
    assert np.array_equal(got.token_ids.cpu().numpy(), want["token_ids"])
    assert np.array_equal(got.parents.cpu().numpy(), want["parents"])
    assert bool(got.state.done[-1])


# ----------------------------------------------------------------- how far scores may be off

# Half the distance below which the order of two beams is settled in 64 bits: what the scan's log-sum may
# be off by.  (The tolerance at the top counts a row's maximum for a wave's, and its errors one by one.)
SCAN_ERROR = 2.0 ** -20


def check_scores(x, C):
    """Totals around zero, so that a score's own rounding hides nothing, of groups of one beam, where no
    near tie has a log-sum formed again."""
    lse = torch.logsumexp(x.double(), dim=-1)
    scores = (lse - x.double().amax(-1)).float().view(-1, 1)
    got = beam_search_select(x, scores, C)
    ids, parents, want = oracle.select(rows_of(x, 1), scores.cpu().numpy(), C)
    assert np.array_equal(got.token_ids.cpu().numpy(), ids)
    assert np.array_equal(got.parents.cpu().numpy(), parents)
    bar = SCAN_ERROR + 2.0 ** -24 * np.abs(want)
    off = np.abs(got.scores.double().cpu().numpy() - want)
    assert (off <= bar).all(), float((off - bar).max())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("G,V", [(3, 700), (2, 9001), (2, 50257), (16, 151936), (8, 262144)])
def test_scores_of_random_rows(device, dtype, G, V):
    gen = torch.Generator(device=device).manual_seed(V)
    x = torch.randn(G * 2, V, device=device, generator=gen)
    for spread in (0.3, 2.5, 6.0):
        check_scores((x * spread).to(DTYPES[dtype]), 3)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("G,V", [(2, 4096), (16, 151936), (16, 262144), (1, 1 << 20)])
@pytest.mark.parametrize("every", [512, 2048, 1 << 30])
def test_scores_of_rows_at_one_distance(device, dtype, G, V, every):
    """Entries at one distance below the maximum, which there is once in the row, in every 2048 or in
    every 512 columns: the scan's worst rows, at the distances where its exponentials round more coarsely."""
    t = DTYPES[dtype]
    for k, far in enumerate((0.7, 2.78, 4.02, 5.55, 6.3, 8.03, 9.9, 11.1, 13.0, 16.1)):
        top = 0.3 + 0.0123 * k  # a value with all its bits set or not: differences round
        x = torch.full((G * 2, V), top - far, device=device).to(t)
        x[:, 7::every] = top
        x[1::2, 11] = top - 0.01
        check_scores(x, 2)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("far", [3.0, 6.5, 12.0, 20.0])
def test_scores_of_peaked_rows(device, dtype, far):
    """One entry above a row of others around `far` below it."""
    gen = torch.Generator(device=device).manual_seed(int(far))
    for G, V in ((3, 700), (16, 151936)):
        x = torch.randn(G * 2, V, device=device, generator=gen) * 0.5 - far
        x[:, V // 3] = 1.0
        check_scores(x.to(DTYPES[dtype]), 2)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("G,V", [(3, 3), (5, 700), (4, 9001), (4, 151936), (64, 151936)])
def test_scores_of_confident_rows(device, dtype, G, V):
    """One entry has nearly all the mass: its log-probability, close to zero, is good to 2^-18 of itself
    (the terms of the others, 44 or less below it, to 3.4e-6; their partial sums to 3.0e-7)."""
    gen = torch.Generator(device=device).manual_seed(V)
    noise = torch.randn(G, V, device=device, generator=gen)
    for far in (7.0, 9.5, 12.0, 16.5, 20.0, 25.0, 31.0, 40.0):
        for spread in (0.0, 0.7):
            x = noise * spread - far
            x[:, [V // 3 - 1, 0, V - 1][int(far) % 3]] = 0.37
            if V > 8:
                x[:, 5] = -math.inf
                x[:, 6] = -3e4
            x = x.to(DTYPES[dtype])
            got = beam_search_select(x, torch.zeros(G, 1, device=device), 2)
            ids, _, _ = oracle.select(rows_of(x, 1), np.zeros((G, 1)), 2)
            assert np.array_equal(got.token_ids.cpu().numpy(), ids)
            rows = x.double()
            top = rows.amax(-1, keepdim=True)
            rest = torch.where(rows < top, (rows - top).exp(), 0.0).sum(-1)
            want = -torch.log1p(rest)  # of the best token, of which there is one a row
            off = (got.scores[:, 0].double() - want).abs()
            # ... and up to 16 roundings of 64-bit sums between 1 and 2, 2^-53 each
            assert (off <= want.abs() * (2.0 ** -18 + 2.0 ** -24) + 2.0 ** -49).all(), (far, spread)


# ----------------------------------------------------------------- answers of odd states


@pytest.mark.parametrize("T", [8, 5000])
def test_a_running_beam_without_a_recorded_parent_is_its_own(device, T):
    """The last recorded parent outside the group: the beam goes on from its own place."""
    W, L = 5, T - 1
    state = BeamState.new(1, W, T, device)
    gen = torch.Generator(device=device).manual_seed(T)
    state.token_history = torch.randint(0, 99, (1, T, W), device=device, generator=gen,
                                        dtype=torch.int32)
    state.parent_history = torch.arange(W, device=device, dtype=torch.int32).expand(1, T, W).clone()
    state.parent_history[0, L - 1] = torch.tensor([-1, W, 4, 2 ** 31 - 1, -2 ** 31], device=device)
    state.scores = -torch.arange(1, W + 1, device=device, dtype=torch.float32)[None] * L
    state.lengths.fill_(L)
    # a finished hypothesis of a beam outside the group counts as beam 0's
    state.finished_scores[0, 0], state.finished_beams[0, 0] = -0.5, W
    state.finished_token_ids[0, 0], state.finished_lengths[0, 0] = 7, L - 2
    got = beam_search_finish(state)
    assert got.lengths[0].tolist() == [L - 2] + [L] * 4
    h = state.token_history[0]
    assert torch.equal(got.token_ids[0, 0, :L - 3], h[:L - 3, 0]) and got.token_ids[0, 0, L - 3] == 7
    for place, (w, own) in enumerate([(0, 0), (1, 1), (2, 4), (3, 3)], start=1):
        assert torch.equal(got.token_ids[0, place, :L - 1], h[:L - 1, own])
        assert got.token_ids[0, place, L - 1] == h[L - 1, w]
    ids, lengths, scores = oracle.finish(host(state), W, 1.0)
    assert np.array_equal(got.token_ids.cpu().numpy(), ids)
    close(got.scores, scores)


@pytest.mark.parametrize("alpha", [-30.0, -400.0, -1e300])
def test_scores_beyond_fp32_are_still_hypotheses(device, alpha):
    """Penalties that take every score below fp32's lowest value: hypotheses are kept, in order."""
    W, V, T, lowest = 3, 40, 30, -torch.finfo(torch.float32).max
    x = torch.full((W, V), -4.0, device=device)
    x[0, 5], x[1, 5], x[2, 8] = 3.0, 2.0, 4.0
    state = BeamState.new(1, W, T, device)
    state.scores = torch.tensor([[-8.0, -8.5, -8.6]], device=device)
    state.lengths.fill_(19)
    state.parent_history = torch.arange(W, device=device, dtype=torch.int32).expand(1, T, W).clone()
    stop = torch.tensor([5], dtype=torch.int32, device=device)
    step = beam_search_step(x, state, stop_token_ids=stop, length_penalty=alpha)
    # the three best candidates: token 5 of beam 0, 8 of beam 2, 5 of beam 1
    assert state.finished_scores[0].tolist() == [lowest, lowest, -math.inf]
    assert state.finished_beams[0].tolist() == [0, 1, -1]
    assert state.finished_lengths[0].tolist() == [20, 20, 0]
    assert step.parents[0, 0] == 2 and step.token_ids[0, 0] == 8 and not state.done[0]
    got = beam_search_finish(state, length_penalty=alpha)
    assert got.scores[0].tolist() == [lowest] * 3 and got.lengths[0].tolist() == [20] * 3
    assert got.token_ids[0, :, 19].tolist() == [5, 5, 8]


@pytest.mark.parametrize("alpha", [400.0, 1e300])
def test_scores_that_vanish_are_still_hypotheses(device, alpha):
    W, V = 2, 40
    x = torch.zeros(W, V, device=device)
    state = BeamState.new(1, W, 30, device)
    state.scores = torch.tensor([[0.0, 0.0]], device=device)
    state.lengths.fill_(19)
    stop = torch.tensor([0], dtype=torch.int32, device=device)
    step = beam_search_step(x, state, stop_token_ids=stop, length_penalty=alpha)
    assert state.finished_scores[0].tolist() == [0.0, -math.inf]
    assert state.finished_token_ids[0].tolist() == [0, -1] and step.token_ids[0].tolist() == [1, 2]


# ----------------------------------------------------------------- reorder's reports


def test_reorder_says_what_it_refuses(device):
    parents = torch.tensor([[1, 0]], dtype=torch.int32, device=device)
    x, y, to = (torch.zeros(2, 6, device=device) for _ in range(3))
    with pytest.raises(ValueError, match="names some of the states"):
        reorder_beams([x, y], parents, out=[x, to])
    with pytest.raises(ValueError, match="names some of the states"):
        reorder_beams([x, y], parents, out=[to, y])
    with pytest.raises(ValueError, match="share memory"):
        reorder_beams([x, y], parents, out=[to, to])
    with pytest.raises(ValueError, match="share memory"):
        reorder_beams([x, y], parents, out=[y, x])
    base = torch.zeros(2, 12, device=device)
    with pytest.raises(ValueError, match="another row stride"):
        reorder_beams(base[:, :6], parents, out=base.view(4, 6)[:2])
    with pytest.raises(RuntimeError):  # more than a call takes
        reorder_beams([torch.zeros(2, 1, device=device) for _ in range(513)], parents)
    assert not any(t.any() for t in (x, y, to, base))


# ----------------------------------------------------------------- steps beside other calls


def test_threads_of_steps_and_selections_on_one_stream(device):
    """Steps and selections of different sizes from several threads: scratch is not mixed up."""
    import threading

    gen = torch.Generator(device=device).manual_seed(5)
    stop = torch.tensor([3], dtype=torch.int32, device=device)
    work = []
    for k, (G, W, V) in enumerate(((3, 4, 30011), (2, 8, 9001), (5, 2, 50257))):
        x = torch.randn(G * W, V, device=device, generator=gen) * 2.5
        state = random_state(device, G, W, 6, k)
        state.lengths.fill_(2)
        out = clone(state)
        out.token_history, out.parent_history = state.token_history, state.parent_history

        def step(x=x, state=state, out=out):
            got = beam_search_step(x, state, stop_token_ids=stop, out=out)
            return got.token_ids, got.parents, out.scores, out.finished_scores

        def select(x=x, scores=state.scores):
            got = beam_search_select(x, scores, 16)
            return got.token_ids, got.parents, got.scores

        work += [(step, [t.clone() for t in step()]), (select, select())]
    torch.cuda.synchronize(device)
    wrong = []

    def run(call, want):
        for _ in range(100):
            if not all(torch.equal(a, b) for a, b in zip(call(), want)):
                wrong.append(call.__name__)

    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# Exponents of length penalties: length ** alpha is formed to 2^-50 and, for an exponent y of two, |y| 2^-52
# of itself (y's own rounding), a quotient is rounded once.
ALPHAS = [0.6, -0.5, 1.7, 2.0, -1.0, 0.001, 8.3]


@pytest.mark.parametrize("alpha", ALPHAS)
@pytest.mark.parametrize("T", [3, 1000, 70001])
def test_scores_of_answers_at_any_exponent(device, alpha, T):
    """Running beams of every length up to 1000, and of lengths around the powers of two up to T."""
    lengths = list(range(1, min(T, 1000) + 1))
    lengths += [n + d for n in 2 ** np.arange(10, 17) for d in (-1, 0, 1) if n + d <= T]
    G = len(lengths)
    if T > 1000:  # histories of T steps a group: a few groups at a time
        lengths = lengths[-21:] + [T]
        G = len(lengths)
    state = BeamState.new(G, 2, T, device)
    r = np.random.default_rng(T)
    scores = -r.uniform(0.1, 300.0, (G, 2)).astype(np.float32)
    state.scores = torch.tensor(scores, device=device)
    state.lengths = torch.tensor(lengths, dtype=torch.int32, device=device)
    got = beam_search_finish(state, length_penalty=alpha)
    want = scores.astype(np.float64) / np.array(lengths, np.float64)[:, None] ** alpha
    want = -np.sort(-want, axis=1)
    off = np.abs(got.scores.double().cpu().numpy() - want)
    # one rounding to fp32, and the power's beside those of numpy's.  70001 ** 8.3 takes scores below 2^-126,
    # where fp32 numbers are 2^-149 apart: a rounding is off by up to 2^-150 however small they are
    power = 2.0 ** -49 + 2.0 ** -52 * np.abs(alpha * np.log2(np.array(lengths, np.float64)))[:, None]
    assert (off <= np.abs(want) * (2.0 ** -24 + power) + 2.0 ** -150).all()
    assert np.array_equal(got.lengths.cpu().numpy(), np.repeat(np.array(lengths)[:, None], 2, axis=1))


@pytest.mark.parametrize("alpha", ALPHAS)
def test_steps_at_any_exponent(device, alpha):
    """Finished hypotheses' scores and the done flags that follow from them."""
    G, W, V, T = 40, 3, 600, 60
    gen = torch.Generator(device=device).manual_seed(1)
    x = torch.randn(G * W, V, device=device, generator=gen) * 2.5
    x[::2, 7] = 9.0
    state = random_state(device, G, W, T, 4)
    check_step(x, state, [7], alpha)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_totals_below_fp32_are_still_candidates(device, dtype):
    """Tokens whose log-probability is below fp32's range: beams with the lowest score, not none."""
    W, V, T, lowest = 2, 40, 4, -torch.finfo(torch.float32).max
    x = torch.full((W, V), -3e38, device=device).to(DTYPES[dtype])
    x[:, 3] = 3e38
    got = beam_search_select(x, torch.tensor([[0.0, -1.0]], device=device), 4)
    assert got.token_ids[0].tolist() == [3, 3, 0, 1] and got.parents[0].tolist() == [0, 1, 0, 0]
    assert got.scores[0].tolist() == [0.0, -1.0, lowest, lowest]
    state = BeamState.new(1, W, T, device)
    step = beam_search_step(x, state)
    assert step.token_ids[0].tolist() == [3, 0] and state.scores[0].tolist() == [0.0, lowest]
    step = beam_search_step(x, state, stop_token_ids=torch.tensor([3], dtype=torch.int32,
                                                                  device=device))
    # the stop token ends both beams, and what goes on is below fp32 again
    assert state.finished_scores[0].tolist() == [0.0, lowest / 2] and bool(state.done[0])
    assert step.parents[0].tolist() == [0, 0] and state.scores[0].tolist() == [lowest, lowest]
