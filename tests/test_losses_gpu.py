"""Training losses on rows of logits against the 64-bit oracle (oracle/losses.py).

Bounds.  An exponent y = (x - M) log2(e) / T carries three roundings, 3 * 2^-24 |y|; a term's relative
error is ln 2 times that, 1.6e-5 at |y| = 126, below which 2^y is 0, and 5e-6 at |y| = 40, beyond which
a term of a row's sum does not count; exp2 is good to 2^-23; a lane adds up to 160 terms, then trees of
ten, which for terms of one sign is at most 170 * 2^-24 = 1e-5.  So a sum is good to 1.6e-5, a
probability to REL = 3.2e-5 of itself.  The log-odds against a token are log s + (M - x) / T, good to
1.6e-5 and to 2^-22 of |M - x| / T (below 40 where the odds are not extreme) and log s: LP = 3e-5 in all.
A log-probability -log(1 + e^odds) changes by 1 - p times that, and has a few ulps of its own.  Entropies
are sums of such values times at most log V.  A gradient is rounded to its dtype once: half a step."""

import math
import threading

import numpy as np
import pytest
import torch

from mvsd.sample import (BeamSearch, Sampler, SamplingMetadata, distillation_loss, policy_loss,
                         preference_loss, token_logprobs)
from mvsd.worker.gpu.sample.logprob import compute_topk_scores
from oracle import losses as oracle

pytestmark = pytest.mark.gpu

REL, LP = 3.2e-5, 3e-5
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
DT = list(DTYPES)


def host(t):
    return t.detach().double().cpu().numpy()


def lp_bound(lp):
    lp = np.asarray(lp, np.float64)
    with np.errstate(invalid="ignore"):
        return np.where(np.isfinite(lp), LP * -np.expm1(lp) + 2.0 ** -21 * np.abs(lp), 0.0)


def close(got, want, bar):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    off = np.abs(got - want)[fine] - np.broadcast_to(bar, want.shape)[fine]
    assert (off <= 0).all(), f"off by {off.max()} beyond the bound"


def close_gradient(got, want, error):
    """`error`: the bound before the rounding to the gradient's dtype."""
    info = torch.finfo(got.dtype)
    bar = error + info.eps / 2 * (np.abs(want) + error) + info.smallest_normal * info.eps
    if got.dtype != torch.float16:
        bar = bar + info.smallest_normal  # below it values may be flushed
    close(host(got), want, bar)


def make(device, shape, dtype, seed, spread=3.0, masked=0.0):
    gen = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(shape, device=device, generator=gen) * spread
    if masked:
        x.masked_fill_(torch.rand(shape, device=device, generator=gen) < masked, -math.inf)
    return x.to(DTYPES[dtype])


def leaf(x):
    return x.detach().requires_grad_()


# --------------------------------------------------------------------------- log-probabilities


def check_logprobs(x, tokens, T=1.0, entropy=False, seed=0):
    x = leaf(x)
    V = x.shape[-1]
    out = token_logprobs(x, tokens, temperature=T, return_entropy=entropy)
    outs = list(out) if entropy else [out]
    rows, ids = host(x).reshape(-1, V), tokens.reshape(-1).cpu().numpy()
    r = np.random.default_rng(seed)
    ups = [torch.tensor(r.normal(size=ids.shape), dtype=torch.float32,
                        device=x.device).view(tokens.shape) for _ in outs]
    grad, = torch.autograd.grad(outs, x, ups)
    assert grad.dtype == x.dtype and grad.shape == x.shape
    want = np.zeros((2, len(ids)))
    slope, bar = np.zeros(rows.shape), np.zeros(rows.shape)
    for n, i in enumerate(ids):
        if i < 0:
            continue
        want[0, n], want[1, n], logp = oracle.token_row(rows[n], i, T)
        if np.isnan(want[0, n]):
            want[1, n] = np.nan
            slope[n] = np.nan
            continue
        g = float(ups[0].reshape(-1)[n])
        gH = float(ups[1].reshape(-1)[n]) if entropy else 0.0
        slope[n], bar[n] = oracle.token_gradient(logp, i, g, gH, T)
    close(host(outs[0]).reshape(-1), want[0], lp_bound(want[0]))
    if entropy:
        close(host(outs[1]).reshape(-1), want[1], LP * (1 + math.log(V)))
    got = grad.reshape(-1, V)
    close_gradient(got, slope, bar * REL * (2 if entropy else 1))
    return outs, grad


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("V", [1, 2, 3, 7, 8, 9, 63, 255, 256, 1000, 2047, 2048, 2049, 8191, 8193])
def test_logprobs_sizes(device, dtype, V):
    x = make(device, (5, V), dtype, V)
    tokens = torch.tensor([0, V - 1, V // 2, -1, V // 3], dtype=torch.int32, device=device)
    check_logprobs(x, tokens, 0.7, entropy=True)
    check_logprobs(x, tokens.long())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("N,V", [(1, 50257), (3, 151936), (40, 32000), (300, 32001), (1100, 5003)])
@pytest.mark.parametrize("entropy", [False, True])
def test_logprobs_rows(device, dtype, N, V, entropy):
    x = make(device, (N, V), dtype, N + V, masked=0.2)
    tokens = torch.randint(0, V, (N,), device=device, dtype=torch.int32,
                           generator=torch.Generator(device=device).manual_seed(1))
    tokens[N // 2] = -1 if N > 1 else tokens[0]
    check_logprobs(x, tokens, entropy=entropy)


@pytest.mark.parametrize("dtype", DT)
def test_logprobs_of_confident_rows(device, dtype):
    """1 - p down to 1e-30 and up to 1 - 1e-30."""
    V = 4001
    x = make(device, (12, V), dtype, 5, spread=0.5)
    x[:, 7] = torch.tensor([8, 12, 16, 20, 30, 40, 60, 80, -10, -30, -60, -80], device=device).to(x.dtype)
    check_logprobs(x, torch.full((12,), 7, dtype=torch.int32, device=device), entropy=True)


@pytest.mark.parametrize("dtype", DT)
def test_masked_and_extreme_rows(device, dtype):
    V, inf = 700, math.inf
    low = torch.finfo(DTYPES[dtype]).min
    x = make(device, (12, V), dtype, 6)
    x[0, 1:] = -inf            # the token alone
    x[1] = -inf                # nothing
    x[2, 5] = inf
    x[3, 5] = math.nan
    x[4, :] = low              # masked by the lowest value throughout
    x[5, 1:] = low
    x[6, 0] = -inf             # the token is masked
    x[7, :] = 0.0
    x[8, 0] = inf              # the token itself
    x[9, 0] = math.nan
    x[10] = math.nan           # left out
    x[11, :350] = -low         # and its opposite
    tokens = torch.zeros(12, dtype=torch.int32, device=device)
    tokens[10] = -1
    for T in (1.0, 0.5):
        if T != 1.0:
            x[11] = 0
            x[4] = 0
            x[5, 1:] = -inf
        y = leaf(x)
        lp = token_logprobs(y, tokens, temperature=T)
        grad, = torch.autograd.grad(lp.sum(), y)
        rows = host(x)
        for n in range(12):
            want = 0.0 if n == 10 else oracle.token_row(rows[n], 0, T)[0]
            close(host(lp[n]), want, lp_bound(want))
            if np.isnan(want):
                assert torch.isnan(grad[n]).all()
            elif n == 10:
                assert (grad[n] == 0).all()
            else:
                slope, bar = oracle.token_gradient(oracle.log_softmax(rows[n], T), 0, 1.0, 0.0, T)
                close_gradient(grad[n], slope, bar * REL)


def test_tokens_outside_the_vocabulary(device):
    x = leaf(make(device, (4, 100), "fp32", 7))
    tokens = torch.tensor([3, 100, 2 ** 40, -2 ** 40], device=device)
    lp = token_logprobs(x, tokens)
    assert torch.isnan(lp).tolist() == [False, True, True, False] and lp[3] == 0
    grad, = torch.autograd.grad(lp[torch.tensor([0, 3])].sum(), x, retain_graph=True)
    assert torch.isfinite(grad[0]).all() and (grad[1:] == 0).all()  # no upstream, no gradient


# --------------------------------------------------------------------------- distillation


def teacher_of(x, K, seed, sampled=False, gaps=0.0):
    """Top entries of a teacher near the rows, shuffled padding, the sampled token in front."""
    r = np.random.default_rng(seed)
    rows = host(x).reshape(-1, x.shape[-1])
    N, V = rows.shape
    ids, values = np.full((N, K), -1, np.int64), np.zeros((N, K), np.float32)
    for n in range(N):
        t = oracle.log_softmax(np.where(np.isfinite(rows[n]), rows[n], -60) + r.normal(size=V))
        k = min(K - (1 if sampled else 0), V)
        top = np.argsort(-t)[:k]
        if sampled:
            top = np.append(r.choice(V), top)
        ids[n, : len(top)], values[n, : len(top)] = top, t[top]
        ids[n, r.random(K) < gaps] = -1
    return (torch.tensor(ids, device=x.device, dtype=torch.int32).view(*x.shape[:-1], K),
            torch.tensor(values, device=x.device).view(*x.shape[:-1], K))


def check_distill(x, ids, teacher, how="forward", tail=True, T=1.0, weights=None, reduction="mean",
                  up=1.0):
    x = leaf(x)
    V, K = x.shape[-1], ids.shape[-1]
    loss = distillation_loss(x, ids, teacher, divergence=how, tail=tail, temperature=T,
                             weights=weights, reduction=reduction)
    N = ids.numel() // K
    up = torch.full_like(loss, up) if reduction != "none" else \
        torch.linspace(0.5, 2.0, N, device=x.device).view(loss.shape)
    grad, = torch.autograd.grad(loss, x, up)
    rows = host(x).reshape(-1, V)
    got = [oracle.distill_row(rows[n], ids.reshape(-1, K)[n].cpu().numpy(),
                              host(teacher).reshape(-1, K)[n], how, tail, T) for n in range(N)]
    w = np.ones(N) if weights is None else host(weights).reshape(-1)
    w = w * np.array([g is not None for g in got])
    f = oracle.mean_factor(w, reduction)
    slope, bar = np.zeros(rows.shape), np.zeros(rows.shape)
    values, sizes = np.zeros(N), np.zeros(N)
    ups = host(up).reshape(-1) if reduction == "none" else np.full(N, host(up))
    for n, g in enumerate(got):
        if g is None or w[n] == 0:
            continue
        values[n], sizes[n] = g[0] * f[n], abs(f[n]) * (3e-5 * g[2])
        slope[n], bar[n] = g[1] * f[n] * ups[n], g[3] * abs(f[n] * ups[n])
    if reduction == "none":
        close(host(loss).reshape(-1), values, sizes + 2.0 ** -22 * np.abs(values))
    else:
        close(host(loss), values.sum(), sizes.sum() + 2.0 ** -20 * np.abs(values).sum())
    close_gradient(grad.reshape(-1, V), slope, bar * 1.5 * REL)
    return loss, grad


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("V,K", [(1, 1), (2, 1), (5, 5), (9, 4), (300, 300), (1000, 64), (2051, 257),
                                 (4099, 512), (8191, 1), (8193, 33)])
@pytest.mark.parametrize("how,tail", [("forward", True), ("forward", False), ("reverse", True),
                                      ("js", True)])
def test_distillation_sizes(device, dtype, V, K, how, tail):
    x = make(device, (4, V), dtype, V * 3 + K)
    ids, teacher = teacher_of(x, K, V + K)
    check_distill(x, ids, teacher, how, tail, 0.9)


@pytest.mark.parametrize("how,tail", [("forward", True), ("forward", False), ("reverse", True),
                                      ("js", True)])
@pytest.mark.parametrize("N,V,dtype", [(1, 151936, "bf16"), (20, 50257, "fp16"), (270, 32000, "bf16"),
                                       (1050, 4001, "fp32")])
def test_distillation_rows(device, N, V, dtype, how, tail):
    x = make(device, (N, V), dtype, N)
    ids, teacher = teacher_of(x, 21, N, sampled=True, gaps=0.1)
    if N > 4:
        ids[3] = -1
    check_distill(x, ids, teacher, how, tail, up=0.5)
    w = torch.rand(N, device=device) + 0.1
    w[0] = 0.0 if N > 1 else w[0]
    check_distill(x, ids.long(), teacher, how, tail, weights=w)
    check_distill(x, ids, teacher, how, tail, weights=w, reduction="sum", up=3.0)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_distillation_of_token_pairs_and_padding(device, reduction):
    """An id may stand in a row many times; padding may stand anywhere."""
    x = make(device, (3, 4, 50), "fp32", 9)
    ids = torch.randint(-3, 6, (3, 4, 40), device=device, dtype=torch.int32,
                        generator=torch.Generator(device=device).manual_seed(2))
    teacher = make(device, (3, 4, 40), "fp32", 10, spread=1.0) - 4.0
    for how, tail in (("forward", True), ("forward", False), ("reverse", True), ("js", True)):
        check_distill(x, ids, teacher, how, tail, reduction=reduction)


def test_distillation_masked_rows(device):
    x = make(device, (8, 600), "bf16", 11, masked=0.6)
    x[:, :8] = make(device, (8, 8), "bf16", 12)
    ids = torch.arange(8, device=device, dtype=torch.int32).expand(8, 8).contiguous()
    teacher = torch.log_softmax(make(device, (8, 9), "fp32", 13), dim=1)[:, :8].contiguous()
    x[0, 8:] = -math.inf       # no mass in the rest: an infinite forward divergence
    teacher[1, 3] = -math.inf  # an entry of no mass
    x[3] = math.nan            # left out
    ids[3] = -1
    teacher[3] = math.nan
    rows = [i for i in range(8) if i != 0]
    for how in ("forward", "js"):
        check_distill(x[rows].contiguous(), ids[rows].contiguous(), teacher[rows].contiguous(), how)
    check_distill(x[2:].contiguous(), ids[2:].contiguous(), teacher[2:].contiguous(), "reverse")
    got = distillation_loss(x, ids, teacher, reduction="none")
    assert got[0] == math.inf and got[3] == 0
    assert distillation_loss(x, ids, teacher, divergence="reverse", reduction="none")[1] == math.inf
    ids[5, 2] = 600
    got = distillation_loss(x, ids, teacher, reduction="none")
    assert torch.isnan(got).nonzero().flatten().tolist() == [5]


# --------------------------------------------------------------------------- policy


def check_policy(x, tokens, old, A, ref=None, low=0.2, high=0.2, kl=0.0, ent=0.0, T=1.0, weights=None,
                 reduction="mean", up=1.0):
    x = leaf(x)
    V = x.shape[-1]
    got = policy_loss(x, tokens, old, A, ref_logprobs=ref, clip_low=low, clip_high=high, kl_coef=kl,
                      entropy_coef=ent, temperature=T, weights=weights, reduction=reduction)
    N = tokens.numel()
    ups = torch.full_like(got.loss, up) if reduction != "none" else \
        torch.linspace(0.5, 2.0, N, device=x.device).view(got.loss.shape)
    grad, = torch.autograd.grad(got.loss, x, ups)
    ups = host(ups).reshape(-1) if reduction == "none" else np.full(N, host(ups))
    rows, ids = host(x).reshape(-1, V), tokens.reshape(-1).cpu().numpy()
    flat = [None if t is None else host(t).reshape(-1) for t in (old, A, ref, weights)]
    w = (np.ones(N) if flat[3] is None else flat[3]) * (ids >= 0)
    f = oracle.mean_factor(w, reduction)
    values, sizes, lps, Hs, kls = (np.zeros(N) for _ in range(5))
    kl_bar = np.zeros(N)
    slope, bar = np.zeros(rows.shape), np.zeros(rows.shape)
    for n, i in enumerate(ids):
        if w[n] == 0:
            continue
        lps[n], Hs[n], logp = oracle.token_row(rows[n], i, T)
        more = (None if old is None else flat[0][n], flat[1][n], None if ref is None else flat[2][n],
                low, high, kl, ent)
        value, c, kls[n], size = oracle.policy_value(lps[n], Hs[n], *more)
        off = lp_bound(lps[n]) + 2.0 ** -22 * (abs(lps[n]) + abs(more[0] or 0) + abs(more[2] or 0))
        around = [oracle.policy_value(lps[n] + d, Hs[n], *more) for d in (-off, off)]
        dc = max(abs(a[1] - c) for a in around) + 2.0 ** -21 * size
        kl_bar[n] = max(abs(a[2] - kls[n]) for a in around) + 2.0 ** -21 * kls[n] + 2.0 ** -40
        values[n] = value * f[n]
        sizes[n] = abs(f[n]) * (max(abs(a[0] - value) for a in around) + 2.0 ** -21 * size
                                + abs(ent) * LP * (1 + math.log(V)))
        g, gH = c * f[n] * ups[n], -ent * f[n] * ups[n]
        slope[n], bar[n] = oracle.token_gradient(logp, i, g, gH, T)
        bar[n] = bar[n] * 2 * REL + oracle.token_gradient(logp, i, dc * f[n] * ups[n], 0.0, T)[1]
    if reduction == "none":
        close(host(got.loss).reshape(-1), values, sizes)
    else:
        close(host(got.loss), values.sum(), sizes.sum() + 2.0 ** -20 * np.abs(values).sum())
    close(host(got.logprobs).reshape(-1), lps, lp_bound(lps))
    if ent:
        close(host(got.entropy).reshape(-1), Hs, LP * (1 + math.log(V)))
    else:
        assert got.entropy is None
    if ref is not None:
        close(host(got.kl).reshape(-1), kls, kl_bar)
    else:
        assert got.kl is None
    close_gradient(grad.reshape(-1, V), slope, bar)
    return got, grad


def policy_inputs(device, lead, V, dtype, seed, spread=0.4):
    x = make(device, (*lead, V), dtype, seed)
    gen = torch.Generator(device=device).manual_seed(seed + 1)
    tokens = torch.randint(0, V, lead, device=device, generator=gen, dtype=torch.int32)
    lp = torch.log_softmax(x.double(), dim=-1).gather(-1, tokens[..., None].long())[..., 0]
    old = (lp + spread * torch.randn(lead, device=device, generator=gen)).float()
    ref = (lp + spread * torch.randn(lead, device=device, generator=gen)).float()
    return x, tokens, old, torch.randn(lead, device=device, generator=gen), ref


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("N,V", [(1, 1), (1, 100), (3, 2049), (5, 8193), (33, 32000), (300, 4099),
                                 (1030, 1003)])
@pytest.mark.parametrize("ent", [0.0, 0.02])
def test_policy(device, dtype, N, V, ent):
    x, tokens, old, A, ref = policy_inputs(device, (N,), V, dtype, N + V)
    if N > 2:
        tokens[1] = -1
    check_policy(x, tokens, old, A, ent=ent)
    check_policy(x, tokens.long(), old, A, ref, 0.1, 0.3, 0.2, ent, T=0.8, up=0.25)
    w = torch.rand(N, device=device)
    w[N // 2] = 0.0 if N > 1 else w[0]
    check_policy(x, tokens, None, A, ref, kl=0.1, ent=ent, weights=w, reduction="sum")
    check_policy(x, tokens, old, A, ref, kl=0.1, ent=ent, weights=w, reduction="none")


@pytest.mark.parametrize("N,V", [(1, 3), (127, 255), (512, 100), (513, 100), (700, 255), (128, 255)])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_policy_of_short_rows(device, N, V, reduction):
    """Rows of one chunk, with their weights added by whom it concerns and by a launch of its own."""
    x, tokens, old, A, ref = policy_inputs(device, (N,), V, "bf16", N + V)
    tokens[N // 3] = -1 if N > 1 else tokens[0]
    w = torch.rand(N, device=device) + 0.5
    check_policy(x, tokens, old, A, ref, kl=0.1, ent=0.01, weights=w, reduction=reduction)
    check_policy(x, tokens, old, A, reduction=reduction)


def test_policy_clips(device):
    """Every side of the clip for both signs; a zero advantage; a border itself."""
    V = 64
    x = make(device, (8, V), "fp32", 21)
    tokens = torch.arange(8, device=device, dtype=torch.int32)
    lp = torch.log_softmax(x.double(), dim=1).gather(1, tokens[:, None].long())[:, 0]
    gap = torch.tensor([0.5, 0.5, -0.5, -0.5, 0.05, -0.05, 0.5, 0.0], device=device)
    A = torch.tensor([1.0, -1.0, 1.0, -1.0, 1.0, -1.0, 0.0, 2.0], device=device)
    old = (lp - gap).float()
    _, grad = check_policy(x, tokens, old, A)
    assert [bool((grad[n] == 0).all()) for n in range(8)] == [True, False, False, True, False, False,
                                                             True, False]
    zero = torch.zeros(2, device=device)
    y = leaf(torch.tensor([[0.0, -math.inf], [0.0, -math.inf]], device=device))
    at = torch.zeros(2, dtype=torch.int32, device=device)
    got = policy_loss(y, at, zero, torch.tensor([1.0, -1.0], device=device), clip_low=0.0,
                      clip_high=0.0, reduction="none")
    assert got.loss.tolist() == [-1.0, 1.0]  # a ratio of 1 at a clip of no width


def test_policy_with_nothing_left(device):
    x, _, old, A, ref = policy_inputs(device, (6,), 500, "bf16", 22)
    x[2] = math.nan
    none = torch.full((6,), -1, dtype=torch.int32, device=device)
    got, grad = check_policy(x, none, old, A, ref, kl=0.1, ent=0.1)
    assert got.loss == 0 and (grad == 0).all()
    tokens = torch.zeros(6, dtype=torch.int32, device=device)
    w = torch.zeros(6, device=device)
    w[1] = 2.0
    keep = w > 0
    got = policy_loss(leaf(x), tokens, old, A, weights=w)
    again = policy_loss(leaf(x), tokens, old, A, weights=keep)  # a mask
    assert torch.isfinite(got.loss) and torch.equal(got.loss, again.loss)


# --------------------------------------------------------------------------- preference


def check_preference(x, tokens, ref, cu=None, beta=0.1, kind="sigmoid", smooth=0.0, margin=0.0,
                     average=False, T=1.0, weights=None, reduction="mean", up=1.0):
    x = leaf(x)
    V = x.shape[-1]
    got = preference_loss(x, tokens, ref, cu_num_tokens=cu, beta=beta, loss_type=kind,
                          label_smoothing=smooth, margin=margin, average=average, temperature=T,
                          weights=weights, reduction=reduction)
    rows, ids = host(x).reshape(-1, V), tokens.reshape(-1).cpu().numpy()
    if cu is None:
        S, L = x.shape[0], x.shape[1]
        spans = [(s * L, (s + 1) * L) for s in range(S)]
    else:
        ends = cu.cpu().numpy()
        S = len(ends)
        spans = [(0 if s == 0 else ends[s - 1], ends[s]) for s in range(S)]
    B = S // 2
    ups = torch.full_like(got.loss, up) if reduction != "none" else \
        torch.linspace(0.5, 2.0, B, device=x.device)
    grad, = torch.autograd.grad(got.loss, x, ups)
    ups = host(ups) if reduction == "none" else np.full(B, host(ups))
    logps = [oracle.token_row(rows[n], i, T) if i >= 0 else (0.0, 0.0, None) for n, i in enumerate(ids)]
    sums, offs, units = np.zeros(S), np.zeros(S), np.ones(S)
    for s, (a, b) in enumerate(spans):
        lps = np.array([logps[n][0] for n in range(a, b)])
        count = sum(ids[n] >= 0 for n in range(a, b))
        units[s] = 1 / max(count, 1) if average else 1.0
        sums[s] = lps.sum() * units[s] if b > a else 0.0
        offs[s] = (lp_bound(lps).sum() + 2.0 ** -22 * np.abs(lps).sum()) * units[s] if b > a else 0.0
    close(host(got.logprobs), sums, offs)
    gain = sums - (host(ref) if ref is not None else 0.0)
    m = gain[:B] - gain[B:]
    off = offs[:B] + offs[B:] + 2.0 ** -22 * (np.abs(gain[:B]) + np.abs(gain[B:])) + \
        (0 if ref is None else 2.0 ** -23 * (np.abs(host(ref)[:B]) + np.abs(host(ref)[B:])))
    w = np.ones(B) if weights is None else host(weights)
    f = oracle.mean_factor(w, reduction)
    values, sizes = np.zeros(B), np.zeros(B)
    slope, bar = np.zeros(rows.shape), np.zeros(rows.shape)
    for i in range(B):
        if w[i] == 0:
            continue
        value, c = oracle.pair_value(m[i], kind, beta, margin, smooth)
        around = [oracle.pair_value(m[i] + d, kind, beta, margin, smooth) for d in (-off[i], off[i])]
        values[i] = value * f[i]
        sizes[i] = abs(f[i]) * (max(abs(a[0] - value) for a in around) + 2.0 ** -21 * (abs(value) + 1))
        dc = max(abs(a[1] - c) for a in around) + 2.0 ** -21 * beta
        for s, sign in ((i, 1.0), (i + B, -1.0)):
            for n in range(*spans[s]):
                if ids[n] < 0:
                    continue
                g = sign * c * units[s] * f[i] * ups[i]
                slope[n], bar[n] = oracle.token_gradient(logps[n][2], ids[n], g, 0.0, T)
                bar[n] = bar[n] * 2 * REL + oracle.token_gradient(
                    logps[n][2], ids[n], dc * units[s] * f[i] * ups[i], 0.0, T)[1]
    if reduction == "none":
        close(host(got.loss), values, sizes)
    else:
        close(host(got.loss), values.sum(), sizes.sum() + 2.0 ** -20 * np.abs(values).sum())
    close_gradient(grad.reshape(-1, V), slope, bar)
    return got, grad


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "squared"])
@pytest.mark.parametrize("average", [False, True])
def test_preference_packed(device, dtype, kind, average):
    """Ragged sequences, two of them empty, rows behind the last."""
    lengths = [5, 0, 17, 1, 9, 30, 2, 0]
    cu = torch.tensor(np.cumsum(lengths), dtype=torch.int32, device=device)
    N, V = sum(lengths) + 4, 2057
    x = make(device, (N, V), dtype, 31)
    x[-1] = math.nan  # behind the last sequence, left out
    tokens = torch.randint(0, V, (N,), device=device, dtype=torch.int32,
                           generator=torch.Generator(device=device).manual_seed(3))
    tokens[[2, 6, 40, N - 1]] = -1
    ref = make(device, (8,), "fp32", 32, spread=5.0) - 100.0
    if average:
        ref = ref * 0.05
    w = torch.tensor([1.0, 0.5, 0.0, 2.0], device=device)
    smooth = 0.1 if kind == "sigmoid" else 0.0
    check_preference(x, tokens, ref, cu, kind=kind, average=average)
    check_preference(x, tokens, None, cu, 0.3, kind, smooth, 0.2, average, 0.9, w, up=0.5)
    check_preference(x, tokens, ref, cu, 0.3, kind, smooth, average=average, weights=w,
                     reduction="none")
    check_preference(x, tokens.long(), ref, cu, 0.05, kind, average=average, reduction="sum")


@pytest.mark.parametrize("shape", [(2, 1, 1), (2, 3, 100), (6, 40, 513), (4, 300, 260)])
def test_preference_padded(device, shape):
    x = make(device, shape, "bf16", 33)
    tokens = torch.randint(-1, shape[2], shape[:2], device=device,
                           generator=torch.Generator(device=device).manual_seed(4))
    tokens[0] = -1  # a sequence of no tokens
    ref = make(device, shape[:1], "fp32", 34) - 6.0 * shape[1]
    check_preference(x, tokens, ref)
    check_preference(x, tokens, ref, average=True, kind="squared", beta=0.5)


@pytest.mark.parametrize("B", [2048, 2049, 5000])
@pytest.mark.parametrize("weighted", [False, True])
def test_many_pairs(device, B, weighted):
    """Whose weights are added once for all of them.  Between the inputs and a value lie at most 20 roundings
    in the sum of the weights, 20 in that of the losses (20 terms a thread, 8 levels of a tree, within a bound
    of 2^-24 each) and 24 others: 2^-18, of which the bars are twice; and a margin is off by four bounds of a
    log-probability."""
    V, beta = 9, 0.2
    x = leaf(make(device, (2 * B, 1, V), "fp32", 35))
    gen = torch.Generator(device=device).manual_seed(36)
    tokens = torch.randint(0, V, (2 * B, 1), device=device, generator=gen)
    w = torch.rand(B, device=device, generator=gen) + 0.1 if weighted else None
    got = preference_loss(x, tokens, beta=beta, weights=w)
    grad, = torch.autograd.grad(got.loss, x)
    y = leaf(x.detach().double())
    lp = torch.log_softmax(y, -1).gather(-1, tokens[..., None])[:, 0, 0]
    f = torch.ones(B, device=device, dtype=torch.float64) if w is None else w.double()
    f = f / f.sum()
    loss = (f * torch.nn.functional.softplus(-beta * (lp[:B] - lp[B:]))).sum()
    slope, = torch.autograd.grad(loss, y)
    off = float(np.max(lp_bound(host(lp.detach()))))
    assert abs(float(got.loss) - float(loss)) <= 2.0 ** -17 * float(loss) + 4 * beta * off
    bar = beta * f.repeat(2)[:, None, None] * (2.0 ** -17 + 4 * beta * off + 2 * off)
    assert ((grad.double() - slope).abs() <= bar).all()


def test_preference_far_margins(device):
    """Margins of thousands: neither overflow nor a lost gradient."""
    x = make(device, (4, 3, 50), "fp32", 35)
    tokens = torch.zeros(4, 3, dtype=torch.int32, device=device)
    for far in (3000.0, -3000.0):
        ref = torch.tensor([far, 0.0, 0.0, 0.0], device=device)
        check_preference(x, tokens, ref, beta=1.0)
        check_preference(x, tokens, ref, beta=1.0, kind="hinge")


# --------------------------------------------------------------------------- layouts


@pytest.mark.parametrize("dtype", DT)
def test_layouts(device, dtype):
    """Rows of any stride and alignment, slices of a batch, expanded rows; ids and values with strides."""
    V = 1001
    big = make(device, (3, 7, 2 * V + 9), dtype, 41)
    for x in (big[:, :-1, 3:V + 3], big[:, 1:, 1:V + 1], big[0, ::2, 5:V + 5], big[::2, 2, :V],
              big.transpose(0, 1)[1:, :, :V], big[1:2, 2:3, :V].expand(2, 3, V)):
        lead = x.shape[:-1]
        gen = torch.Generator(device=device).manual_seed(5)
        tokens = torch.randint(0, V, (*lead, 2), device=device, generator=gen)[..., 1]
        check_logprobs(x, tokens, entropy=True)
        A = torch.randn((*lead[:-1], 1), device=device, generator=gen)  # one value for a row of tokens
        old = torch.full((), -6.0, device=device)
        y = leaf(x)
        got = policy_loss(y, tokens, old, A)
        want = policy_loss(leaf(x.contiguous()), tokens.contiguous(), old.expand(lead).contiguous(),
                           A.expand(lead).contiguous())
        assert torch.equal(got.loss, want.loss) and torch.equal(got.logprobs, want.logprobs)
        ids, teacher = teacher_of(x, 9, 42)
        check_distill(x, ids, teacher)


def test_gradients_of_broadcast_rows(device):
    """One row used many times: its gradient is the sum."""
    V = 300
    row = leaf(make(device, (1, V), "fp32", 43))
    tokens = torch.arange(6, device=device)
    token_logprobs(row.expand(6, V), tokens).sum().backward()
    want = sum(oracle.token_gradient(oracle.log_softmax(host(row)[0]), i, 1.0, 0.0)[0]
               for i in range(6))
    close(host(row.grad)[0], want, 6 * (REL + 2.0 ** -23))


def test_offsets_beyond_32_bits(device):
    """Logits and gradients of more than 2^31 entries: the first and the last rows."""
    V, N = 151936, 14300
    x = torch.zeros(N, V, dtype=torch.bfloat16, device=device)
    ends = torch.tensor([0, 1, N - 2, N - 1], device=device)
    x[ends] = make(device, (4, V), "bf16", 44)
    tokens = torch.full((N,), -1, dtype=torch.int32, device=device)
    tokens[ends] = torch.tensor([5, V - 1, 0, 77], dtype=torch.int32, device=device)
    y = leaf(x)
    got = policy_loss(y, tokens, None, torch.ones(N, device=device), reduction="sum")
    grad, = torch.autograd.grad(got.loss, y)
    for n in ends.tolist():
        lp, _, logp = oracle.token_row(host(x[n]), int(tokens[n]), 1.0)
        close(host(got.logprobs[n]), lp, lp_bound(lp))
        slope, bar = oracle.token_gradient(logp, int(tokens[n]), -1.0, 0.0)
        close_gradient(grad[n], slope, bar * REL)
    assert int((grad[2:N - 2] != 0).sum()) == 0


@pytest.mark.parametrize("lead", [(0,), (0, 5), (4, 0)])
def test_no_rows(device, lead):
    x = leaf(torch.zeros(*lead, 30, device=device, dtype=torch.bfloat16))
    tokens = torch.zeros(lead, dtype=torch.int32, device=device)
    v = torch.zeros(lead, device=device)
    ids = torch.zeros(*lead, 3, dtype=torch.int32, device=device)
    for reduction in ("mean", "sum", "none"):
        for loss in (policy_loss(x, tokens, v, v, reduction=reduction).loss,
                     distillation_loss(x, ids, ids.float(), reduction=reduction)):
            assert loss.shape == (lead if reduction == "none" else ())
            assert float(loss.sum()) == 0
            grad, = torch.autograd.grad(loss.sum(), x)
            assert grad.shape == x.shape
    assert token_logprobs(x, tokens).shape == lead
    if len(lead) == 1:
        cu = torch.zeros(4, dtype=torch.int32, device=device)
        got = preference_loss(x, tokens, cu_num_tokens=cu)
        assert abs(float(got.loss) - math.log(2)) < 1e-6 and (got.logprobs == 0).all()
    elif lead[0] == 4:
        assert abs(float(preference_loss(x, tokens).loss) - math.log(2)) < 1e-6


# --------------------------------------------------------------------------- as a program uses them


def calls(device, N=40, V=3001, dtype="bf16", seed=51):
    """Every operator with a scalar loss, as functions of the logits."""
    x, tokens, old, A, ref = policy_inputs(device, (N,), V, dtype, seed)
    ids, teacher = teacher_of(x, 12, seed)
    cu = torch.tensor([N // 4, N // 2, N // 2 + 3, N - 2], dtype=torch.int32, device=device)
    sums = torch.full((4,), -80.0, device=device)
    return x, {
        "logprobs": lambda x: token_logprobs(x, tokens).sum(),
        "entropy": lambda x: sum(v.sum() for v in token_logprobs(x, tokens, return_entropy=True)),
        "distill": lambda x: distillation_loss(x, ids, teacher),
        "js": lambda x: distillation_loss(x, ids, teacher, divergence="js", weights=A.abs()),
        "policy": lambda x: policy_loss(x, tokens, old, A, ref_logprobs=ref, kl_coef=0.1).loss,
        "bonus": lambda x: policy_loss(x, tokens, old, A, entropy_coef=0.1, reduction="sum").loss,
        "preference": lambda x: preference_loss(x, tokens, sums, cu_num_tokens=cu).loss,
    }


SHAPES = [(40, 3001), (600, 5000)]


@pytest.mark.parametrize("N,V", SHAPES)
def test_same_results_again(device, N, V):
    x, ops = calls(device, N, V)
    for name, op in ops.items():
        got = []
        for _ in range(2):
            y = leaf(x)
            loss = op(y)
            got.append((loss.detach(), torch.autograd.grad(loss, y)[0]))
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1]), name
        with torch.no_grad():
            assert torch.equal(op(x), got[0][0]), name


@pytest.mark.parametrize("N,V", SHAPES)
def test_backward_twice_and_scaled(device, N, V):
    """A kept graph gives its gradient again, also after the first one was changed, and for another
    upstream; leaves accumulate."""
    x, ops = calls(device, N, V, "fp32")
    for name, op in ops.items():
        y = leaf(x)
        loss = op(y)
        first, = torch.autograd.grad(loss, y, retain_graph=True)
        kept = first.clone()
        first.zero_()
        second, = torch.autograd.grad(loss, y, retain_graph=True)
        assert torch.equal(second, kept), name
        half, = torch.autograd.grad(loss, y, torch.full_like(loss, -0.5), retain_graph=True)
        tiny = torch.finfo(torch.float32).smallest_normal
        assert ((half - kept * -0.5).abs() <= kept.abs() * 2.0 ** -20 + tiny).all(), name
        zero, = torch.autograd.grad(loss, y, torch.zeros_like(loss), retain_graph=True)
        assert (zero == 0).all(), name
        loss.backward(retain_graph=True)
        loss.backward()
        assert ((y.grad - 2 * kept).abs() <= kept.abs() * 2.0 ** -20 + tiny).all(), name


@pytest.mark.parametrize("N,V", SHAPES)
def test_saved_tensors_that_move(device, N, V):
    """What the backward pass needs may be kept elsewhere and come back to another place."""
    x, ops = calls(device, N, V)
    for name, op in ops.items():
        y, z = leaf(x), leaf(x)
        want, = torch.autograd.grad(op(y), y)
        with torch.autograd.graph.save_on_cpu():
            loss = op(z)
        got, = torch.autograd.grad(loss, z, retain_graph=True)
        assert torch.equal(got, want), name
        again, = torch.autograd.grad(loss, z)
        assert torch.equal(again, want), name


@pytest.mark.parametrize("N,V", SHAPES)
def test_recomputed(device, N, V):
    """Forgotten in the forward pass and formed again in the backward pass."""
    from torch.utils.checkpoint import checkpoint
    x, ops = calls(device, N, V)
    for name, op in ops.items():
        for reentrant in (False, True):
            y, z = leaf(x), leaf(x)
            op(y).backward()
            checkpoint(op, z, use_reentrant=reentrant).backward()
            assert torch.equal(y.grad, z.grad), name


def test_through_a_graph_of_layers(device):
    """The logits are an output of a layer, the loss a term of a sum; other terms use the same logits."""
    h = make(device, (64, 32), "fp32", 61, spread=1.0)
    weight = leaf(make(device, (500, 32), "fp32", 62, spread=0.3))
    tokens = torch.arange(64, device=device)
    A = torch.ones(64, device=device)

    def grads(loss_of):
        logits = h @ weight.t()
        return torch.autograd.grad(loss_of(logits), weight)[0]

    ids = tokens[:, None].int()
    got = grads(lambda x: policy_loss(x, tokens, None, A).loss
                + 0.5 * distillation_loss(x, ids, torch.zeros(64, 1, device=device), tail=False))
    want = grads(lambda x: -1.0 * torch.log_softmax(x, dim=1).gather(1, tokens[:, None]).mean()
                 - 0.5 * torch.log_softmax(x, dim=1).gather(1, tokens[:, None]).mean())
    # the policy's value is -1, its gradient that of -lp; both are means over 64 rows
    scale = (torch.log_softmax(h @ weight.t(), dim=1).exp() / 64).t().abs() @ h.abs()
    assert ((got - want).abs() <= 1e-4 * (scale + h.abs().amax() / 64)).all()


def test_second_derivatives_are_refused(device):
    x, ops = calls(device)
    y = leaf(x.float())
    grad, = torch.autograd.grad(ops["policy"](y), y, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_changed_logits_are_noticed(device):
    x, ops = calls(device, dtype="fp32")
    for name, op in ops.items():
        y = leaf(x) * 1.0
        loss = op(y)
        y.add_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


@pytest.mark.parametrize("N,V", SHAPES)
def test_streams(device, N, V):
    """Calls on another stream, and beside calls on the first."""
    x, ops = calls(device, N, V)
    want = {}
    for name, op in ops.items():
        y = leaf(x)
        loss = op(y)
        want[name] = loss.detach(), torch.autograd.grad(loss, y)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        got = {}
        for name, op in ops.items():
            y = leaf(x)
            loss = op(y)
            got["main " + name] = name, loss.detach(), torch.autograd.grad(loss, y)[0]
            with torch.cuda.stream(side):
                y = leaf(x)
                loss = op(y)
                got["side " + name] = name, loss.detach(), torch.autograd.grad(loss, y)[0]
        torch.cuda.synchronize()
        for what, (name, loss, grad) in got.items():
            assert torch.equal(loss, want[name][0]) and torch.equal(grad, want[name][1]), what


@pytest.mark.parametrize("N,V", SHAPES)
def test_captured_and_replayed(device, N, V):
    """Two graphs over the same memory, eager calls and new logits between their replays."""
    x, ops = calls(device, N, V)
    static = leaf(x.clone())
    graphs = {}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for op in ops.values():  # allocations and the library's first calls
            torch.autograd.grad(op(static), static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for name, op in ops.items():
        for k in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                loss = op(static) * 1.0
                grad, = torch.autograd.grad(loss, static)
            graphs[name, k] = g, loss, grad
    for step in range(3):
        fresh = make(device, x.shape, "bf16", 70 + step)
        with torch.no_grad():
            static.copy_(fresh)
        want = {}
        for name, op in ops.items():
            y = leaf(fresh)
            loss = op(y)
            want[name] = loss.detach(), torch.autograd.grad(loss, y)[0]
        for (name, k), (g, loss, grad) in graphs.items():
            g.replay()
        torch.cuda.synchronize()
        for (name, k), (g, loss, grad) in graphs.items():
            assert torch.equal(loss.detach(), want[name][0]), (name, k, step)
            assert torch.equal(grad, want[name][1]), (name, k, step)


def test_no_host_synchronisation(device):
    x, ops = calls(device)
    for op in ops.values():
        y = leaf(x)
        torch.autograd.grad(op(y), y)
    torch.cuda.synchronize()
    mode = torch.cuda.get_sync_debug_mode()
    torch.cuda.set_sync_debug_mode("error")
    try:
        for op in ops.values():
            y = leaf(x)
            torch.autograd.grad(op(y), y)
    finally:
        torch.cuda.set_sync_debug_mode(mode)


def test_nothing_else_is_written(device):
    """The inputs stay, and so does what lies around the rows."""
    x, tokens, old, A, ref = policy_inputs(device, (30,), 1500, "bf16", 81)
    pool = torch.full((30, 1600), 7.0, device=device, dtype=torch.bfloat16)
    pool[:, 50:1550] = x
    before = [t.clone() for t in (pool, tokens, old, A, ref)]
    y = leaf(pool[:, 50:1550])
    got = policy_loss(y, tokens, old, A, ref_logprobs=ref, kl_coef=0.1)
    torch.autograd.grad(got.loss, y)
    for t, b in zip((pool, tokens, old, A, ref), before):
        assert torch.equal(t, b)


def test_together_with_what_the_framework_gives(device):
    """A serving step's scores, tokens and answers, then the three losses on them."""
    V, N = 2000, 24
    target = make(device, (N, V), "fp32", 91)
    sampled = Sampler(logprobs_mode="raw_logprobs").forward(
        target.clone(), SamplingMetadata(temperature=torch.ones(N, device=device), all_greedy=False,
                                         all_random=True, top_k=None, top_p=None, max_num_logprobs=4))
    tokens = sampled.sampled_token_ids.reshape(-1)
    scores = compute_topk_scores(target, 16, tokens)
    draft = make(device, (N, V), "bf16", 92)
    check_distill(draft, scores.logprob_token_ids, scores.logprobs)
    check_distill(target.bfloat16(), scores.logprob_token_ids, scores.logprobs, "reverse")
    # the sampler's own log-probabilities are those of the policy that drew
    old = sampled.logprobs_tensors.logprobs[:, 0].contiguous()
    close(host(token_logprobs(target, tokens)), host(old), 2 * lp_bound(host(old)))
    ref = token_logprobs(draft, tokens)
    check_policy(target.bfloat16(), tokens, old, torch.randn(N, device=device), ref, kl=0.1)
    # answers of a beam search: the best of each request against its last
    G, W, T = 3, 4, 5
    search = BeamSearch(G, W, T, device)
    for t in range(T):
        search.step(make(device, (G * W, V), "fp32", 93 + t))
    answers = search.finish(W)
    pairs = torch.cat([answers.token_ids[:, 0], answers.token_ids[:, W - 1]])  # [2 G, T], -1 behind
    model = make(device, (2 * G, T, V), "bf16", 99)
    ref = token_logprobs(target[: 2 * G * T // T].repeat_interleave(T, 0).view(2 * G, T, V), pairs)
    check_preference(model, pairs, ref.sum(dim=1))


# --------------------------------------------------------------------------- refusals


def refusals(device):
    x = torch.zeros(4, 10, device=device)
    ids = torch.zeros(4, dtype=torch.int32, device=device)
    v = torch.zeros(4, device=device)
    two, t = ids[:, None].expand(4, 2), v[:, None].expand(4, 2)
    cu = torch.tensor([2, 4], dtype=torch.int32, device=device)
    lp, distill, policy, pref = token_logprobs, distillation_loss, policy_loss, preference_loss
    return [
        (TypeError, lambda: lp(x.double(), ids)), (TypeError, lambda: lp(x[0], ids[0])),
        (ValueError, lambda: lp(x.t(), ids.new_zeros(10))), (ValueError, lambda: lp(x, ids[:3])),
        (TypeError, lambda: lp(x, ids.short())), (NotImplementedError, lambda: lp(x, ids.cpu())),
        (ValueError, lambda: lp(x[:, :0], ids)), (ValueError, lambda: lp(x, ids, temperature=0.0)),
        (ValueError, lambda: lp(x, ids, temperature=math.nan)),
        (ValueError, lambda: distill(x, two[:, :0], t[:, :0])),
        (ValueError, lambda: distill(x, ids[:, None].expand(4, 513), v[:, None].expand(4, 513))),
        (ValueError, lambda: distill(x, two, t[:, :1].expand(4, 3))),
        (ValueError, lambda: distill(x, ids, v)), (TypeError, lambda: distill(x, two, t.half())),
        (ValueError, lambda: distill(x, two, t, divergence="kl")),
        (ValueError, lambda: distill(x, two, t, divergence="js", tail=False)),
        (ValueError, lambda: distill(x, two, t, weights=v[:3])),
        (TypeError, lambda: distill(x, two, t, weights=v.double())),
        (ValueError, lambda: policy(x, ids, v, None)), (TypeError, lambda: policy(x, ids, v.half(), v)),
        (ValueError, lambda: policy(x, ids, v, v, kl_coef=0.1)),
        (ValueError, lambda: policy(x, ids, v, v, clip_low=-0.1)),
        (ValueError, lambda: policy(x, ids, v, v, clip_high=math.inf)),
        (ValueError, lambda: policy(x, ids, v, v, entropy_coef=math.nan)),
        (ValueError, lambda: policy(x, ids, v, v[:2])),
        (ValueError, lambda: pref(x, ids)),
        (ValueError, lambda: pref(x.view(2, 2, 10), ids.view(2, 2), cu_num_tokens=cu)),
        (ValueError, lambda: pref(x, ids, cu_num_tokens=torch.cat([cu, cu[-1:]]))),
        (TypeError, lambda: pref(x, ids, cu_num_tokens=cu.long())),
        (ValueError, lambda: pref(x, ids, v, cu_num_tokens=cu)),
        (ValueError, lambda: pref(x, ids, cu_num_tokens=cu, beta=0.0)),
        (ValueError, lambda: pref(x, ids, cu_num_tokens=cu, loss_type="kto")),
        (ValueError, lambda: pref(x, ids, cu_num_tokens=cu, label_smoothing=1.5)),
        (ValueError, lambda: pref(x, ids, cu_num_tokens=cu, label_smoothing=0.1, loss_type="hinge")),
        (ValueError, lambda: pref(x, ids, cu_num_tokens=cu, weights=v)),
    ]


def test_refusals(device):
    for k, (error, call) in enumerate(refusals(device)):
        with pytest.raises(error):
            call()
            print("accepted:", k)


# --------------------------------------------------------------------------- masked entries

DIVERGENCES = [("forward", True), ("forward", False), ("reverse", True), ("js", True)]


def masked_entries(device, dtype, N, base, T, value=-math.inf):
    """Rows around `base` whose entries have the logit `value`: all of them in every third row (the first
    one among them), two of four in the next, none in the last."""
    x = make(device, (N, 600), dtype, 101, spread=3.0 * min(T, 1.0)).float() + base
    gen = torch.Generator(device=device).manual_seed(102)
    ids = torch.rand((N, 600), device=device, generator=gen).argsort(dim=1)[:, :4].int()
    gone = torch.ones(N, 4, dtype=torch.bool, device=device)
    gone[1::3, 2:] = False
    gone[2::3] = False
    x.scatter_(1, ids.long(), torch.where(gone, value, x.gather(1, ids.long())))
    teacher = torch.log_softmax(make(device, (N, 5), "fp32", 103, spread=1.0), dim=1)[:, :4].contiguous()
    return x.to(DTYPES[dtype]), ids, teacher


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("how,tail", DIVERGENCES)
@pytest.mark.parametrize("N", [3, 100])
def test_distillation_entries_without_mass(device, dtype, how, tail, N):
    """The student gives none of a row's entries any mass; its other logits lie anywhere.  By workgroups that
    share a row, and in one pass."""
    for base, T in ((0.0, 1.0), (-60.0, 1.0), (-110.0, 1.0), (-300.0, 1.0), (300.0, 1.0), (-40.0, 0.3),
                    (-10.0, 0.1), (10.0, 0.1)):
        x, ids, teacher = masked_entries(device, dtype, N, base, T)
        for reduction in ("mean", "none"):
            loss, grad = check_distill(x, ids, teacher, how, tail, T, reduction=reduction)
            assert torch.isfinite(grad).all()
            assert not torch.isnan(loss).any()
            assert bool(torch.isfinite(loss).all()) == (how != "forward")


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("how", ["reverse", "js"])
@pytest.mark.parametrize("N", [3, 100])
def test_distillation_entries_far_below(device, dtype, how, N):
    """Entries of a probability that is 0 in 64 bits too, one of which the teacher rules out: they add nothing
    where the student's mass is the weight."""
    for gap, T in ((1000.0, 1.0), (120.0, 0.1)):
        x, ids, teacher = masked_entries(device, dtype, N, 0.0, T, -gap)
        teacher[:, 1] = -math.inf
        keep = torch.arange(N, device=device) % 3 == 0  # in the others an entry has mass
        loss, grad = check_distill(x, torch.where(keep[:, None], ids, -1), teacher, how, True, T)
        assert torch.isfinite(loss) and torch.isfinite(grad).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("how,tail", DIVERGENCES)
@pytest.mark.parametrize("N", [3, 100])
def test_distillation_entries_masked_by_the_lowest_value(device, dtype, how, tail, N):
    """Over a temperature below 1 it is beyond fp32, as -inf is: the same bits.  (-inf itself against the
    oracle: above.)"""
    low = torch.finfo(DTYPES[dtype]).min
    for T in (0.9, 0.5, 0.01):
        got = []
        for value in (-math.inf, low):
            x, ids, teacher = masked_entries(device, dtype, N, -5.0 * T, T, value)
            x = leaf(x)
            loss = distillation_loss(x, ids, teacher, divergence=how, tail=tail, temperature=T)
            got.append((loss.detach(), torch.autograd.grad(loss, x)[0]))
        assert torch.equal(got[0][0], got[1][0]) and not torch.isnan(got[1][0])
        assert torch.equal(got[0][1], got[1][1]) and torch.isfinite(got[1][1]).all()


def test_distillation_of_what_the_teacher_rules_out(device):
    """Entries without a teacher's mass that the student masks by the lowest value: the tail alone counts."""
    x, ids, _ = masked_entries(device, "fp32", 3, 0.0, 0.5, torch.finfo(torch.float32).min)
    for N in (1, 100):
        y = x[:1].expand(N, -1).contiguous()
        for how in ("forward", "js"):
            teacher = torch.full((N, 4), -math.inf, device=device)
            loss, grad = check_distill(y, ids[:1].expand(N, 4).contiguous(), teacher, how, True, 0.5)
            assert torch.isfinite(loss) and torch.isfinite(grad).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("how,tail", DIVERGENCES)
@pytest.mark.parametrize("N", [7, 100])
def test_distillation_rows_without_a_distribution(device, dtype, how, tail, N):
    """Their values and the whole of their gradients are NaN, whatever else is masked; the other rows' are not."""
    V, inf = 600, math.inf
    x, ids, teacher = masked_entries(device, dtype, N, 0.0, 1.0, -1.0)
    first = ids[:, 0].long()
    bad = x[1:6]
    bad[:4].fill_(-inf)
    bad[1, first[2]] = math.nan
    bad[2, first[3]] = inf
    bad[3, first[4]] = 0.0
    ids[4, 1] = V              # an entry that is no token
    bad[4, 5] = math.nan
    x = leaf(x)
    got = distillation_loss(x, ids, teacher, divergence=how, tail=tail, reduction="none")
    none, = torch.autograd.grad(got.sum(), x)
    each, = torch.autograd.grad(distillation_loss(x, ids, teacher, divergence=how, tail=tail, reduction="sum"), x)
    rows = torch.arange(N, device=device)
    wrong = (rows >= 1) & (rows < 6)
    assert torch.equal(torch.isnan(got), wrong)
    for grad in (none, each):
        assert torch.isnan(grad[wrong]).all() and torch.isfinite(grad[~wrong]).all()


# --------------------------------------------------------------------------- tokens without others


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("V", [1, 2, 300])
def test_a_token_alone_at_any_height(device, dtype, V):
    """Nothing beside it: a log-probability and an entropy of 0, no gradient, also where its logit over the
    temperature is beyond fp32; -inf itself is no distribution.  A mean of 120 values of -1 has the rounding of
    1 / 120 and at most nine of a sum over 256 threads: within 10 * 2^-24 < 2^-20."""
    low = torch.finfo(DTYPES[dtype]).min
    heights = torch.tensor([low, -low, low / 2, 0.0, -1e4, 1e4, -math.inf], device=device).to(DTYPES[dtype])
    N = 140
    for T in (1e-6, 0.5, 1.0, 10.0):
        x = torch.full((N, V), -math.inf, device=device, dtype=DTYPES[dtype])
        x[:, V - 1] = heights.repeat(N // 7)
        nothing = torch.isinf(x[:, V - 1])
        tokens = torch.full((N,), V - 1, device=device)
        y = leaf(x)
        lp, H = token_logprobs(y, tokens, temperature=T, return_entropy=True)
        grad, = torch.autograd.grad([lp, H], y, [torch.ones_like(lp), torch.ones_like(H)])
        for rows in (lp, H, grad):
            assert torch.isnan(rows[nothing]).all() and (rows[~nothing] == 0).all()
        y = leaf(x)
        got = policy_loss(y, tokens, None, torch.ones(N, device=device), entropy_coef=0.1, temperature=T,
                          weights=~nothing)
        grad, = torch.autograd.grad(got.loss, y)
        assert abs(got.loss.item() + 1) <= 2.0 ** -20 and (grad == 0).all()


# --------------------------------------------------------------------------- memory


def test_memory_between_the_passes(device):
    """Recomputation and saved tensors on the host leave nothing of the logits' size on the device, and after a
    backward pass nothing of it is left but the gradient."""
    from torch.utils.checkpoint import checkpoint
    N, V = 600, 5000
    x, ops = calls(device, N, V, "fp32")
    size = x.numel() * 4

    def held(make):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        kept = make()
        return torch.cuda.memory_allocated() - before, kept

    for name, op in ops.items():
        y = leaf(x)
        more, loss = held(lambda: checkpoint(op, y, use_reentrant=False))
        assert more < size / 4, name
        assert held(loss.backward)[0] < size * 1.25, name
        y = leaf(x)
        with torch.autograd.graph.save_on_cpu():
            more, loss = held(lambda: op(y))
        assert more < size / 4, name
        assert held(loss.backward)[0] < size * 1.25, name
        y = leaf(x)
        more, loss = held(lambda: op(y))
        assert more + held(loss.backward)[0] < size * 1.25, name


# --------------------------------------------------------------------------- several threads


@pytest.mark.parametrize("N,V", SHAPES)
def test_threads_go_back_through_one_graph(device, N, V):
    """With no thread of the engine's between them, each with an upstream of its own (powers of two: exact)."""
    x, ops = calls(device, N, V, "fp32")
    for name, op in ops.items():
        y = leaf(x)
        loss = op(y)
        want, = torch.autograd.grad(loss, y, retain_graph=True)
        loss = op(y)
        got, scales = {}, [1.0, 2.0, 0.5, -1.0]

        def back(n):
            with torch.autograd.set_multithreading_enabled(False):
                got[n] = [torch.autograd.grad(loss, y, torch.full_like(loss, scales[n]), retain_graph=True)[0]
                          for _ in range(5)]

        threads = [threading.Thread(target=back, args=(n,)) for n in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        tiny = torch.finfo(torch.float32).smallest_normal
        for n, grads in got.items():
            for grad in grads:
                assert ((grad - scales[n] * want).abs() <= want.abs() * 2.0 ** -20 + 2 * tiny).all(), (name, n)


# --------------------------------------------------------------------------- forward mode


@pytest.mark.parametrize("N,V", SHAPES)
def test_forward_mode_is_refused(device, N, V):
    """With and without a gradient wanted beside it; logits cut from their tangent are taken."""
    import torch.autograd.forward_ad as forward_ad
    x, ops = calls(device, N, V)
    for name, op in ops.items():
        want = op(x)
        with forward_ad.dual_level():
            for y in (x.detach().clone(), leaf(x.clone())):
                dual = forward_ad.make_dual(y, torch.ones_like(x))
                with pytest.raises(NotImplementedError):
                    op(dual)
                with torch.no_grad(), pytest.raises(NotImplementedError):
                    op(dual)
                assert torch.equal(op(dual.detach()), want), name


# --------------------------------------------------------------------------- rows of no pair


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("N,V", [(5, 700), (1500, 300)])
def test_rows_without_pairs(device, reduction, N, V):
    """A packed batch of no sequences with rows behind them."""
    x = leaf(make(device, (N, V), "bf16", 111))
    x.data[0] = math.nan
    tokens = torch.zeros(N, dtype=torch.int32, device=device)
    cu = torch.zeros(0, dtype=torch.int32, device=device)
    got = preference_loss(x, tokens, torch.zeros(0, device=device), cu_num_tokens=cu, reduction=reduction,
                          weights=torch.zeros(0, device=device))
    assert got.logprobs.shape == (0,) and got.loss.shape == ((0,) if reduction == "none" else ())
    assert got.loss.sum().item() == 0
    grad, = torch.autograd.grad(got.loss.sum(), x)
    assert grad.shape == x.shape and (grad == 0).all()


# --------------------------------------------------------------------------- plans of the kernels


@pytest.mark.parametrize("how,tail", DIVERGENCES)
@pytest.mark.parametrize("V,K,dtype", [(256, 512, "fp32"), (256, 512, "bf16"), (257, 64, "fp16"), (1000, 256, "fp32"),
                                       (1000, 130, "bf16"), (4099, 65, "fp32"), (32000, 512, "bf16"),
                                       (32000, 512, "fp32")])
def test_distillation_entries_of_several_waves(device, V, K, dtype, how, tail):
    """In one pass: more entries than a wave has lanes, or than threads hold the row; rows left out, by their
    entries and by their weight; entries of all rows' ends."""
    N = 90
    x = make(device, (N, V), dtype, V + K)
    ids, teacher = teacher_of(x, K, V + K + 1, sampled=True, gaps=0.05)
    ids[:, -1] = V - 1
    ids[1::5] = -1
    w = torch.rand(N, device=device) + 0.1
    w[2::7] = 0.0
    check_distill(x, ids, teacher, how, tail, 0.8, weights=w)
    check_distill(x, ids, teacher, how, tail, weights=w, reduction="sum", up=0.5)


@pytest.mark.parametrize("how", ["forward", "js"])
@pytest.mark.parametrize("V,dtype", [(196608, "bf16"), (196609, "bf16"), (80000, "fp32")])
def test_distillation_of_long_rows(device, V, dtype, how):
    """Columns beyond what a workgroup's registers hold, and one more than those whose entries it marks.  A lane
    adds 192 terms at most, so that a sum is good to 202 * 2^-24 + 5e-6 < 1.8e-5; the bars have 3e-5."""
    N = 81
    x = make(device, (N, V), dtype, V)
    ids, teacher = teacher_of(x[:12], 33, V, sampled=True)
    ids = torch.cat([ids, ids.new_full((N - 12, 33), -1)]).roll(40, 0)
    ids[45, 3], ids[45, 4] = V - 1, V - 8
    teacher = torch.cat([teacher, teacher.new_zeros(N - 12, 33)]).roll(40, 0)
    check_distill(x, ids, teacher, how)


@pytest.mark.parametrize("V,dtype", [(151936, "fp32"), (262144, "bf16"), (262145, "fp16")])
@pytest.mark.parametrize("ent", [0.0, 0.02])
def test_policy_of_long_rows(device, V, dtype, ent):
    """The same of a policy loss, which has no limit there: 256 terms a lane, good to 266 * 2^-24 + 5e-6 < 2.2e-5."""
    N = 130
    x, tokens, old, A, ref = policy_inputs(device, (N,), V, dtype, V)
    keep = torch.arange(N, device=device) % 9 == 0
    tokens[0], tokens[9], tokens[18] = V - 1, 0, V - 9
    old[:19:9] = -13.0
    ref[:19:9] = -12.0
    check_policy(x, torch.where(keep, tokens, -1), old, A, ref, kl=0.1, ent=ent)


@pytest.mark.parametrize("V", [151936, 300000])
def test_logprobs_of_many_long_rows(device, V):
    """A workgroup adds a chunk of up to 2^18 columns: 1024 terms a lane, a sum within 1034 * 2^-24 + 5e-6 < 6.7e-5, a
    log-probability within that and 1e-6, a gradient's term within that and its own exponential's 5e-6."""
    N, bound = 1030, 7.5e-5
    x = torch.zeros(N, V, dtype=torch.bfloat16, device=device)
    live = torch.arange(3, N, 97, device=device)
    x[live] = make(device, (len(live), V), "bf16", V)
    tokens = torch.full((N,), -1, dtype=torch.int32, device=device)
    tokens[live] = torch.randint(0, V, (len(live),), device=device, dtype=torch.int32,
                                 generator=torch.Generator(device=device).manual_seed(7))
    x = leaf(x)
    lp, H = token_logprobs(x, tokens, return_entropy=True)
    grad, = torch.autograd.grad([lp, H], x, [torch.ones_like(lp), torch.full_like(H, 0.5)])
    for n in live.tolist():
        t = int(tokens[n])
        want, entropy, logp = oracle.token_row(host(x[n]), t)
        close(host(lp[n]), want, bound * -np.expm1(want) + 2.0 ** -21 * abs(want))
        close(host(H[n]), entropy, bound * (1 + math.log(V)))
        slope, bar = oracle.token_gradient(logp, t, 1.0, 0.5)
        close_gradient(grad[n], slope, bar * 2 * bound)
    assert (lp[tokens < 0] == 0).all() and (H[tokens < 0] == 0).all()
    assert int(grad[tokens < 0].count_nonzero()) == 0


# --------------------------------------------------------------------------- ratios beyond fp32


@pytest.mark.parametrize("N", [6, 132])
def test_policy_ratios_beyond_fp32(device, N):
    """e^150 times an advantage of 0 is 0, and a positive advantage's ratio is clipped; a NaN stays one."""
    V = 500
    x, tokens, old, _, ref = policy_inputs(device, (N,), V, "fp32", 121)
    old[::2] -= 150.0
    A = torch.tensor([0.0, 0.0, 1.5, -1.0, 0.0, 0.5], device=device).repeat(N // 6)
    for ent in (0.0, 0.02):
        got, grad = check_policy(x, tokens, old, A, ref, kl=0.1, ent=ent)
        assert torch.isfinite(got.loss) and torch.isfinite(grad).all()
        check_policy(x, tokens, old, A, reduction="none", ent=ent)
    x[0, 3] = math.nan
    got = policy_loss(x, tokens, old, A, reduction="none")
    assert torch.isnan(got.loss).nonzero().flatten().tolist() == [0]
    assert torch.isnan(policy_loss(leaf(x), tokens, old, A).loss)
