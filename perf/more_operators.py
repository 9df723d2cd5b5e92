"""Training losses on rows of logits, as measurable cases.

Four operators on rows of logits [N, V], each one pass of what a program does with the tokens and
log-probabilities that the samplers, the verification and beam search give it:

    logprobs    token_logprobs: the log-probabilities (and entropies) of given tokens, as the policy
                and the preference loss need them of an older or a reference model; with gradients
                where they are trained on
    distill     distillation_loss: a draft model against the target's top log-probabilities
    policy      policy_loss: clipped policy loss with a KL term on sampled tokens
    preference  preference_loss: paired log ratios of whole answers

A training pass gives its loss and the gradient of the logits.  ``listed()`` holds the standing
cases, ``draw(rng)`` gives one more of the same ranges.  With ``own`` false a pass is the operator's
plain form, elementary torch operations.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_PACKAGE = str(Path(__file__).resolve().parents[1] / "vllm-from-scratch_amd")
VOCAB = 151936
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
NINF = -math.inf
MOST = 2048 * VOCAB  # entries of the largest case

# --------------------------------------------------------------------------- the cases


def _case(name, kind, N, V, dtype, *, T=1.0, pad=0.0, masked=0.0, beyond=0, **more):
    """N rows of V logits; T: temperature; pad: the share of rows that are left out (prompts,
    padding: token -1); masked: the share of the vocabulary that a grammar rules out (-inf);
    beyond: columns behind the vocabulary in memory (a padded output layer)."""
    return {"name": name, "kind": kind, "N": N, "V": V, "dtype": dtype, "T": T, "pad": pad,
            "masked": masked, "beyond": beyond, **more}


def _logprobs(name, N, V, dtype, *, train=False, entropy=False, **more):
    return _case(name, "logprobs", N, V, dtype, train=train, entropy=entropy, **more)


def _distill(name, N, V, dtype, K, *, how="forward", tail=True, sampled=False, scale=0.0, **more):
    """K teacher tokens a row; how: the divergence; tail: the rest of the vocabulary is an outcome;
    sampled: the sampled token stands before the top ones, as in the scores of the samplers (so it
    mostly stands there twice); scale: weights that carry a loss scale (0: the plain mean)."""
    return _case(name, "distill", N, V, dtype, K=K, how=how, tail=tail, sampled=sampled,
                 scale=scale, **more)


def _policy(name, N, V, dtype, *, old=True, kl=0.0, entropy=0.0, high=0.2, **more):
    """old: tokens of an earlier policy (else of this one); kl, entropy: the terms' coefficients."""
    return _case(name, "policy", N, V, dtype, old=old, kl=kl, entropy=entropy, high=high, **more)


def _preference(name, pairs, L, V, dtype, *, how="sigmoid", packed=True, ref=True, average=False,
                smooth=0.0, **more):
    """Pairs of answers of up to L tokens; packed: one behind the other, a few rows behind the last
    (else [2 * pairs, L, V], padded)."""
    c = _case(name, "preference", 0, V, dtype, pairs=pairs, L=L, how=how, packed=packed, ref=ref,
              average=average, smooth=smooth, **more)
    c["N"] = int(_lengths(c).sum()) + 3 if packed else 2 * pairs * L
    return c


def _lengths(case):
    """The answers' lengths, the same ones for every seed of a case."""
    n, L = 2 * case["pairs"], case["L"]
    made = np.random.default_rng([n, L]).integers(max(1, L // 2), L + 1, size=n)
    made[0] = L
    return made


def listed():
    return [
        # one decoding step of a few requests scored by a second model: the smallest call
        _logprobs("logprobs_step", 4, VOCAB, "bf16"),
        # a batch of rollouts scored by the reference model, prompts left out
        _logprobs("logprobs_score", 2048, VOCAB, "bf16", pad=0.1),
        # log-probabilities and entropies that a user's own loss is built on
        _logprobs("logprobs_train", 1500, 50257, "fp32", train=True, entropy=True, pad=0.1),
        # a draft model tuned while it serves, a few verified tokens at a time
        _distill("distill_online", 16, VOCAB, "bf16", 8),
        # an ordinary batch, the target's scores as the samplers return them
        _distill("distill_scores", 1024, VOCAB, "bf16", 33, sampled=True, beyond=64),
        # mode-seeking, a small draft vocabulary, fp16 with its loss scale
        _distill("distill_reverse", 4096, 32000, "fp16", 20, how="reverse", scale=4096.0, T=0.8),
        # many teacher tokens a row, over those alone
        _distill("distill_wide", 2048, VOCAB, "bf16", 128, tail=False, pad=0.05),
        # one short answer: the smallest policy update
        _policy("policy_answer", 24, 32000, "bf16", old=False),
        # a full batch with the KL term to a reference: the largest
        _policy("policy_batch", 2048, VOCAB, "bf16", kl=0.05, high=0.28, pad=0.1),
        # fp32 rows under a grammar, entropy bonus
        _policy("policy_entropy", 2000, 32001, "fp32", entropy=0.01, masked=0.3, T=0.9),
        # a pair of short answers
        _preference("preference_pair", 1, 40, 32000, "bf16"),
        # a packed batch of pairs, prompts left out
        _preference("preference_batch", 16, 64, VOCAB, "bf16", pad=0.2, smooth=0.1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["logprobs", "distill", "distill", "policy", "policy", "preference"])
    V = VOCAB if rng.random() < 0.3 else _log_int(rng, 1000, VOCAB)
    if V != VOCAB:
        V = V | 1 if rng.random() < 0.5 else V // 64 * 64
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    N = _log_int(rng, 1, min(8192, MOST * 2 // (V * SIZE[dtype])))
    more = {"T": rng.choice([1.0, 1.0, 0.7, 1.5]), "pad": rng.choice([0.0, 0.0, 0.1, 0.5]),
            "masked": rng.choice([0.0, 0.0, 0.0, 0.5, 0.95]),
            "beyond": rng.choice([0, 0, 1, 64, 1000])}
    if kind == "logprobs":
        c = _logprobs("", N, V, dtype, train=rng.random() < 0.6, entropy=rng.random() < 0.5, **more)
    elif kind == "distill":
        how = rng.choice(["forward", "forward", "reverse", "js"])
        c = _distill("", N, V, dtype, _log_int(rng, 1, 256), how=how,
                     tail=how != "forward" or rng.random() < 0.6, sampled=rng.random() < 0.4,
                     scale=1024.0 if dtype == "fp16" else rng.choice([0.0, 0.0, 8.0]), **more)
    elif kind == "policy":
        c = _policy("", N, V, dtype, old=rng.random() < 0.8, kl=rng.choice([0.0, 0.05, 0.5]),
                    entropy=rng.choice([0.0, 0.0, 0.01]), high=rng.choice([0.2, 0.28]), **more)
    else:
        more["pad"] = min(more["pad"], 0.3)
        L = _log_int(rng, 4, 1024)
        pairs = _log_int(rng, 1, max(1, N // (2 * L)))
        if 2 * pairs * L * V * SIZE[dtype] > 2 * MOST:
            L = max(4, MOST // (pairs * V * SIZE[dtype]))
        c = _preference("", pairs, L, V, dtype, how=rng.choice(["sigmoid", "sigmoid", "hinge",
                                                                "squared"]),
                        packed=rng.random() < 0.6, ref=rng.random() < 0.8,
                        average=rng.random() < 0.3, smooth=rng.choice([0.0, 0.0, 0.1]), **more)
    del c["name"]
    return c


def _left_out(case):
    """Which rows are left out, the same ones for every seed of a case."""
    N = case["N"]
    if case["kind"] != "preference":
        out = np.zeros(N, bool)
        out[np.random.default_rng([N, 7]).permutation(N)[: int(N * case["pad"])]] = True
        return out
    out = np.ones(N, bool)
    at = 0
    for b, length in enumerate(_lengths(case)):
        start = at if case["packed"] else b * case["L"]
        out[start + int(length * case["pad"]): start + length] = False  # behind the prompt
        at += length
    return out


def work(case):
    N, V, size = case["N"], case["V"], SIZE[case["dtype"]]
    rows = N - int(_left_out(case).sum())
    train = case["kind"] != "logprobs" or case["train"]
    small = N * 16 + (N * case["K"] * 8 if case["kind"] == "distill" else 0)
    # an entry: its part of the maximum and of the sum of exponentials; its exponential again and
    # its product for the gradient
    return {"bytes": (rows + (N if train else 0)) * V * size + small,
            "flops": rows * V * (5 + (4 if train else 0))}


# --------------------------------------------------------------------------- inputs


class _Rng:
    """Host and device generators made from one seed."""

    def __init__(self, seed):
        self.device = torch.device("cuda", torch.cuda.current_device())
        self.host = np.random.default_rng(seed)
        self.gen = torch.Generator(device=self.device).manual_seed(seed)

    def put(self, values, dtype=torch.float32):
        return torch.as_tensor(np.ascontiguousarray(values), device=self.device).to(dtype)

    def normal(self, *shape):
        return torch.randn(shape, device=self.device, generator=self.gen)

    def ids(self, V, *shape):
        return torch.randint(0, V, shape, device=self.device, generator=self.gen)


def _row_logprobs(case, x, tokens):
    """What the model gives the tokens, some rows at a time."""
    got = []
    for a in range(0, x.shape[0], 256):
        y = x[a:a + 256].double() / case["T"]
        got.append(y.gather(1, tokens[a:a + 256, None])[:, 0] - y.logsumexp(dim=1))
    return torch.cat(got)


def prepare(case, seed):
    r = _Rng(seed)
    s = dict(case)
    kind, N, V = case["kind"], case["N"], case["V"]
    rest = torch.empty(N, V + case["beyond"], device=r.device)
    rest.normal_(generator=r.gen).mul_(2.0)  # what is not likely
    x = rest[:, :V]
    if case["masked"]:
        gone = torch.rand((N, V), device=r.device, generator=r.gen) < case["masked"]
        x.masked_fill_(gone, NINF)
        del gone
    # the most likely tokens stand out of the rest: by about its log-sum-exp
    top = math.log(V) + 2.0
    left_out = r.put(_left_out(case), torch.bool)
    if kind == "distill":
        K = case["K"]
        gaps = torch.randint(1, V // K + 1, (N, K), device=r.device, generator=r.gen)
        ids = gaps.cumsum(dim=1) - 1
        ids = ids.gather(1, torch.rand((N, K), device=r.device, generator=r.gen).argsort(dim=1))
        height = top + 1.0 - 1.2 * torch.arange(K, device=r.device).float().sqrt()
        teacher = (height + 0.5 * r.normal(N, K)).sort(dim=1, descending=True).values
        x.scatter_(1, ids, teacher + 0.5 * r.normal(N, K))
        rest_mass = torch.full((N, 1), top, device=r.device)
        teacher = teacher - torch.cat([teacher, rest_mass], dim=1).logsumexp(dim=1, keepdim=True)
        if case["sampled"]:
            # the sampled token is one of the top ones or, now and then, none of them
            at = (torch.rand((N, 1), device=r.device, generator=r.gen) ** 2 * K).long()
            other = r.ids(V, N, 1)
            is_top = torch.rand((N, 1), device=r.device, generator=r.gen) < 0.9
            is_top |= (ids == other).any(dim=1, keepdim=True)
            ids = torch.cat([torch.where(is_top, ids.gather(1, at), other), ids], dim=1)
            teacher = torch.cat([torch.where(is_top, teacher.gather(1, at), -16.0), teacher], dim=1)
        s["ids"] = ids.masked_fill(left_out[:, None], -1)
        s["teacher"] = teacher
        s["weights"] = None
        if case["scale"]:
            s["weights"] = (0.5 + torch.rand(N, device=r.device, generator=r.gen)) * case["scale"] / N
    else:
        tokens = r.ids(V, N)
        x.scatter_(1, tokens[:, None], top + 2.0 * r.normal(N, 1))
    # the logits as the output layer leaves them
    buffer = rest.to(DTYPES[case["dtype"]])
    del rest
    x = buffer[:, :V]
    if kind == "preference":
        B, n = case["pairs"], _lengths(case)
        lp = _row_logprobs(case, x, tokens).masked_fill(left_out, 0.0)
        if case["packed"]:
            cu = r.put(np.cumsum(n), torch.int32)
            owner = r.put(np.append(np.repeat(np.arange(2 * B), n), [2 * B] * 3), torch.long)
        else:
            cu = None
            owner = torch.arange(2 * B, device=r.device).repeat_interleave(case["L"])
            x = buffer.view(2 * B, case["L"], V + case["beyond"])[:, :, :V]
        sums = torch.zeros(2 * B + 1, dtype=torch.float64, device=r.device)
        sums.index_add_(0, owner, lp)
        s["ref"] = (sums[: 2 * B] + 4.0 * r.normal(2 * B)).float() if case["ref"] else None
        s["cu"], s["owner"] = cu, owner
    if kind == "policy":
        lp = _row_logprobs(case, x, tokens)
        # log ratios of a few steps of learning, none of them a rounding away from the clip's border
        gap = 0.2 * r.normal(N).double()
        for border in (0.8, 1.0 + case["high"]):
            gap = torch.where((gap.exp() - border).abs() < 1e-3, gap + 0.01, gap)
        s["old"] = (lp - gap).float() if case["old"] else None
        s["ref"] = (lp + 0.3 * r.normal(N)).float() if case["kl"] else None
        s["advantages"] = r.normal(N)
    if kind == "logprobs":
        s["upstream"] = r.normal(2, N) / N
    if kind != "distill":
        tokens = tokens.masked_fill(left_out, -1)
        s["tokens"] = tokens.view(x.shape[:-1]).int()
    train = kind != "logprobs" or case["train"]
    s["logits"] = x.detach().requires_grad_(train and own)
    return s


# --------------------------------------------------------------------------- the plain forms


def _first_places(ids):
    """Entries that count: no padding, and a token's first place in its row."""
    K = ids.shape[1]
    before = torch.ones(K, K, dtype=torch.bool, device=ids.device).tril(-1)
    twice = torch.cat([((part[:, :, None] == part[:, None, :]) & before).any(dim=2)
                       for part in ids.split(1 << 8)])
    return (ids >= 0) & ~twice


def _log_softmax_plain(s):
    y = s["logits"].detach().reshape(-1, s["V"]).float() / s["T"]
    y = y - y.amax(dim=1, keepdim=True)
    return y - y.exp().sum(dim=1, keepdim=True).log()


def _token_gradient_plain(s, logp, tokens, c, entropy=None):
    """c (onehot - p) / T, and the entropy's part with its own factor, in the logits' type."""
    p = logp.exp()
    grad = p * -c[:, None]
    if entropy is not None:
        H, cH = entropy
        grad = grad - torch.where(p > 0, cH[:, None] * p * (logp + H[:, None]), 0.0)
    grad.scatter_add_(1, tokens[:, None], c[:, None])
    return (grad / s["T"]).to(s["logits"].dtype)


def _entropy_plain(logp):
    return -torch.where(logp > NINF, logp.exp() * logp, 0.0).sum(dim=1)


def _mean_factor(w):
    total = w.sum()
    return w / torch.where(total == 0, 1.0, total)


def _logprobs_plain(s):
    logp = _log_softmax_plain(s)
    tokens = s["tokens"].reshape(-1).long()
    keep = tokens >= 0
    tokens = tokens.clamp(min=0)
    lp = logp.gather(1, tokens[:, None])[:, 0].masked_fill(~keep, 0.0)
    out = {"logprobs": lp}
    H = None
    if s["entropy"]:
        H = _entropy_plain(logp).masked_fill(~keep, 0.0)
        out["entropy"] = H
    if s["train"]:
        up = s["upstream"] * keep
        out["grad"] = _token_gradient_plain(s, logp, tokens, up[0],
                                            (H, up[1]) if s["entropy"] else None)
    return out


def _distill_plain(s):
    logp = _log_softmax_plain(s)
    ids, V = s["ids"].long(), s["V"]
    use = _first_places(ids)
    at = ids.clamp(min=0)
    row = use.any(dim=1)
    teacher = s["teacher"].masked_fill(~use, NINF)
    lp = logp.gather(1, at)
    if s["tail"]:
        q, logq = teacher.exp(), teacher
        # the rest of the vocabulary; no finer than what fp32 log-probabilities resolve
        qt = (1.0 - teacher.double().exp().sum(dim=1, keepdim=True)).float().clamp(min=2.0 ** -24)
        others = logp.scatter(1, torch.where(use, at, at[:, :1]), NINF)
        top = others.amax(dim=1, keepdim=True).clamp(min=-1e30)
        lt = top + (others - top).exp().sum(dim=1, keepdim=True).log()
        del others
        q, logq, lp = (torch.cat(pair, dim=1) for pair in ((q, qt), (logq, qt.log()), (lp, lt)))
        use = torch.cat([use, row[:, None]], dim=1)
    else:
        logq = teacher / s["T"]
        logq = logq - logq.logsumexp(dim=1, keepdim=True)
        q = logq.exp()
    p = lp.exp()
    zero = torch.zeros((), device=p.device)
    if s["how"] == "forward":
        loss = torch.where(use & (q > 0), q * (logq - lp), zero)
        pD = -q
    elif s["how"] == "reverse":
        loss = torch.where(use & (p > 0), p * (lp - logq), zero)
        pD = loss
    else:
        m = torch.log(0.5 * (p + q))
        kl_p = torch.where(use & (p > 0), p * (lp - m), zero)
        loss = 0.5 * (torch.where(use & (q > 0), q * (logq - m), zero) + kl_p)
        pD = 0.5 * kl_p
    pD = torch.where(use, pD, zero)
    loss = loss.sum(dim=1)
    w = row.float() if s["weights"] is None else s["weights"] * row
    f = _mean_factor(w) if s["weights"] is None else w
    total = (torch.where(row, loss, zero) * f).sum()
    # gradient: p_j (D - sum of p D), D that of j's outcome
    mean = pD.sum(dim=1, keepdim=True)
    rest = -mean
    if s["tail"]:
        rest = rest + torch.where(p[:, -1:] > 0, pD[:, -1:] / p[:, -1:], zero)
    top = (pD - p * mean)[:, : ids.shape[1]]
    grad = logp.exp_() * rest
    # places that do not count write what the first one writes
    first = use[:, : ids.shape[1]].float().argmax(dim=1, keepdim=True)
    same = use[:, : ids.shape[1]]
    grad.scatter_(1, torch.where(same, at, at.gather(1, first)),
                  torch.where(same, top, top.gather(1, first)))
    grad = torch.where(row[:, None], grad * (f[:, None] / s["T"]), zero)
    return {"loss": total, "grad": grad.to(s["logits"].dtype)}


def _policy_plain(s):
    logp = _log_softmax_plain(s)
    tokens = s["tokens"].reshape(-1).long()
    keep = tokens >= 0
    tokens = tokens.clamp(min=0)
    f = _mean_factor(keep.float())
    lp = logp.gather(1, tokens[:, None])[:, 0]
    A = s["advantages"]
    ratio = (lp - s["old"]).exp() if s["old"] is not None else torch.ones_like(lp)
    free, bound = ratio * A, ratio.clamp(0.8, 1.0 + s["high"]) * A
    loss = -torch.minimum(free, bound)
    c = torch.where(free <= bound, -free, 0.0)
    out = {}
    if s["kl"]:
        d = s["ref"] - lp
        kl = d.exp() - d - 1.0
        loss = loss + s["kl"] * kl
        c = c + s["kl"] * (1.0 - d.exp())
        out["kl"] = kl.masked_fill(~keep, 0.0)
    entropy = None
    if s["entropy"]:
        H = _entropy_plain(logp)
        loss = loss - s["entropy"] * H
        entropy = (H, -s["entropy"] * f)
        out["entropy"] = H.masked_fill(~keep, 0.0)
    out["loss"] = (loss * f).sum()
    out["logprobs"] = lp.masked_fill(~keep, 0.0)
    out["grad"] = _token_gradient_plain(s, logp, tokens, c * f, entropy)
    return out


BETA = 0.1


def _preference_plain(s):
    logp = _log_softmax_plain(s)
    tokens = s["tokens"].reshape(-1).long()
    B, keep = s["pairs"], tokens >= 0
    tokens = tokens.clamp(min=0)
    lp = logp.gather(1, tokens[:, None])[:, 0].masked_fill(~keep, 0.0)
    sums = torch.zeros(2 * B + 1, device=lp.device).index_add_(0, s["owner"], lp)[: 2 * B]
    unit = torch.ones(2 * B, device=lp.device)
    if s["average"]:
        n = torch.zeros(2 * B + 1, device=lp.device).index_add_(0, s["owner"], keep.float())
        unit = 1.0 / n[: 2 * B].clamp(min=1.0)
        sums = sums * unit
    gain = sums - s["ref"] if s["ref"] is not None else sums
    m = gain[:B] - gain[B:]
    h, e = BETA * m, s["smooth"]
    if s["how"] == "sigmoid":
        soft = torch.log1p((-h.abs()).exp())
        loss = (1.0 - e) * (soft + (-h).clamp(min=0)) + e * (soft + h.clamp(min=0))
        c = BETA * (e / (1.0 + (-h).exp()) - (1.0 - e) / (1.0 + h.exp()))
    elif s["how"] == "hinge":
        loss = (1.0 - h).clamp(min=0)
        c = torch.where(h < 1.0, -BETA, 0.0)
    else:
        off = m - 0.5 / BETA
        loss, c = off * off, 2.0 * off
    c = torch.cat([c, -c]) / B * unit
    c = torch.cat([c, c.new_zeros(1)])[s["owner"]] * keep
    grad = _token_gradient_plain(s, logp, tokens, c)
    return {"loss": loss.mean(), "logprobs": sums, "grad": grad.view(s["logits"].shape)}


# --------------------------------------------------------------------------- the framework's calls


def _framework():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import mvsd.sample

    return mvsd.sample


def _own(s):
    ops = _framework()
    x, kind = s["logits"], s["kind"]
    if kind == "logprobs":
        got = ops.token_logprobs(x, s["tokens"], temperature=s["T"], return_entropy=s["entropy"])
        out = {"logprobs": got}
        if s["entropy"]:
            out = dict(zip(("logprobs", "entropy"), got))
        if s["train"]:
            outs = list(out.values())
            out["grad"], = torch.autograd.grad(outs, x, list(s["upstream"][: len(outs)]))
        return {k: v.detach() for k, v in out.items()}
    if kind == "distill":
        loss = ops.distillation_loss(x, s["ids"], s["teacher"], divergence=s["how"],
                                     tail=s["tail"], temperature=s["T"], weights=s["weights"],
                                     reduction="mean" if s["weights"] is None else "sum")
        return {"loss": loss.detach(), "grad": torch.autograd.grad(loss, x)[0]}
    if kind == "policy":
        got = ops.policy_loss(x, s["tokens"], s["old"], s["advantages"], ref_logprobs=s["ref"],
                              clip_high=s["high"], kl_coef=s["kl"], entropy_coef=s["entropy"],
                              temperature=s["T"])
        out = {"loss": got.loss.detach(), "logprobs": got.logprobs}
        if s["kl"]:
            out["kl"] = got.kl
        if s["entropy"]:
            out["entropy"] = got.entropy
        out["grad"], = torch.autograd.grad(got.loss, x)
        return out
    got = ops.preference_loss(x, s["tokens"], s["ref"], cu_num_tokens=s["cu"], beta=BETA,
                              loss_type=s["how"],
                              label_smoothing=s["smooth"] if s["how"] == "sigmoid" else 0.0,
                              average=s["average"], temperature=s["T"])
    return {"loss": got.loss.detach(), "logprobs": got.logprobs,
            "grad": torch.autograd.grad(got.loss, x)[0]}


def run(state):
    if own:
        return _own(state)
    return {"logprobs": _logprobs_plain, "distill": _distill_plain, "policy": _policy_plain,
            "preference": _preference_plain}[state["kind"]](state)


# --------------------------------------------------------------------------- in 64 bits


def _blocks(N, V):
    step = max(1, (1 << 27) // V)
    return [slice(a, min(N, a + step)) for a in range(0, N, step)]


def _softmax_exact(s, rows):
    x = s["logits"].detach().reshape(-1, s["V"])[rows].double() / s["T"]
    return x - torch.logsumexp(x, dim=1, keepdim=True)


def _token_exact(s, tokens, make):
    """Per row log-probabilities and entropies; then the gradient for the factors of `make`."""
    N, V = tokens.numel(), s["V"]
    keep = tokens >= 0
    at = tokens.clamp(min=0)[:, None]
    lp = torch.zeros(N, dtype=torch.float64, device=tokens.device)
    H = torch.zeros_like(lp)
    for b in _blocks(N, V):
        logp = _softmax_exact(s, b)
        lp[b] = logp.gather(1, at[b])[:, 0]
        H[b] = torch.special.entr(logp.exp()).sum(dim=1)
    c, cH = make(lp, H)
    grad = torch.zeros(N, V, dtype=torch.float64, device=tokens.device)
    for b in _blocks(N, V):
        logp = _softmax_exact(s, b)
        p = logp.exp()
        g = torch.zeros_like(p).scatter_(1, at[b], 1.0).sub_(p).mul_(c[b, None])
        if cH is not None:
            g += cH[b, None] * (torch.special.entr(p) - p * H[b, None])
        grad[b] = g / s["T"] * keep[b, None]
    return lp * keep, H * keep, grad


def _distill_exact(s):
    ids, V = s["ids"].long(), s["V"]
    N, K = ids.shape
    row = (ids >= 0).any(dim=1)
    w = row.double() if s["weights"] is None else s["weights"].double() * row
    f = w / w.sum() if s["weights"] is None and bool(row.any()) else w
    total = torch.zeros((), dtype=torch.float64, device=ids.device)
    grad = torch.zeros(N, V, dtype=torch.float64, device=ids.device)
    for b in _blocks(N, V):
        logp = _softmax_exact(s, b)
        part, n = ids[b], logp.shape[0]
        # a token's outcome: its first place in the row, or K, the tail
        outcome = torch.full((n, V), K, dtype=torch.long, device=ids.device)
        r = torch.arange(n, device=ids.device)
        counts = torch.zeros(n, K + 1, dtype=torch.bool, device=ids.device)
        for k in range(K - 1, -1, -1):
            there = part[:, k] >= 0
            outcome[r[there], part[there, k]] = k
        for k in range(K):
            there = part[:, k] >= 0
            counts[r[there], k] = outcome[r[there], part[there, k]] == k
        v = s["teacher"][b].double()
        v = torch.where(counts[:, :K], v, NINF)
        logq = torch.full((n, K + 1), NINF, dtype=torch.float64, device=ids.device)
        if s["tail"]:
            logq[:, :K] = v
            logq[:, K] = (1.0 - v.exp().sum(dim=1)).clamp(min=2.0 ** -24).log()
            counts[:, K] = True
        else:
            logq[:, :K] = torch.log_softmax(v / s["T"], dim=1)
        lp = torch.full((n, K + 1), NINF, dtype=torch.float64, device=ids.device)
        lp[:, :K] = logp.gather(1, part.clamp(min=0))
        top = torch.where(outcome == K, logp, NINF)
        lp[:, K] = torch.logsumexp(top, dim=1)
        del top
        p, q = lp.exp(), logq.exp()
        if s["how"] == "forward":
            terms = torch.where(q > 0, q * (logq - lp), 0.0)
            D = torch.where(p > 0, -q / p, 0.0)
        elif s["how"] == "reverse":
            terms = torch.where(p > 0, p * (lp - logq), 0.0)
            D = torch.where(p > 0, lp - logq, 0.0)
        else:
            m = ((p + q) / 2).log()
            terms = torch.where(q > 0, q * (logq - m), 0.0) / 2
            terms = terms + torch.where(p > 0, p * (lp - m), 0.0) / 2
            D = torch.where(p > 0, lp - m, 0.0) / 2
        terms, D = torch.where(counts, terms, 0.0), torch.where(counts, D, 0.0)
        total += torch.where(row[b], terms.sum(dim=1) * f[b], 0.0).sum()
        mean = (torch.where(counts, p, 0.0) * D).sum(dim=1, keepdim=True)
        g = logp.exp_() * (D.gather(1, outcome) - mean) * (f[b, None] / s["T"])
        grad[b] = torch.where(row[b, None], g, 0.0)
    return {"loss": total, "grad": grad}


def exact(case, seed):
    if case["N"] * case["V"] > MOST * 1.01 or case.get("K", 0) * case["N"] > 1 << 20:
        return None
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "distill":
        return _distill_exact(s)
    tokens = s["tokens"].reshape(-1).long()
    keep = (tokens >= 0).double()
    out = {}
    if kind == "logprobs":
        up = s["upstream"].double()
        lp, H, grad = _token_exact(s, tokens, lambda lp, H: (up[0], up[1] if s["entropy"] else None))
        out["logprobs"] = lp
        if s["entropy"]:
            out["entropy"] = H
        if s["train"]:
            out["grad"] = grad
        return out
    if kind == "policy":
        f = keep / keep.sum().clamp(min=1)
        A = s["advantages"].double()
        low, high = float(np.float32(0.8)), float(np.float32(1.0 + s["high"]))

        def make(lp, H):
            r = (lp - s["old"].double()).exp() if s["old"] is not None else torch.ones_like(lp)
            clipped = torch.where(A >= 0, r > high, r < low)
            loss = -torch.where(clipped, r.clamp(low, high), r) * A
            c = torch.where(clipped, 0.0, -r * A)
            if s["kl"]:
                d = s["ref"].double() - lp
                out["kl"] = (torch.expm1(d) - d) * keep
                loss, c = loss + s["kl"] * out["kl"], c - s["kl"] * torch.expm1(d)
            if s["entropy"]:
                loss = loss - s["entropy"] * H
            out["loss"] = (loss * f).sum()
            return c * f, -s["entropy"] * f if s["entropy"] else None

        lp, H, grad = _token_exact(s, tokens, make)
        if s["entropy"]:
            out["entropy"] = H
        out["logprobs"], out["grad"] = lp, grad
        return out
    B = case["pairs"]

    def make(lp, H):
        total = lp.new_zeros(2 * B + 1).index_add_(0, s["owner"], lp * keep)[: 2 * B]
        n = lp.new_zeros(2 * B + 1).index_add_(0, s["owner"], keep)[: 2 * B].clamp(min=1)
        unit = 1 / n if s["average"] else torch.ones_like(n)
        total = total * unit
        out["logprobs"] = total.clone()
        total.requires_grad_()
        with torch.enable_grad():
            gain = total if s["ref"] is None else total - s["ref"].double()
            m = gain[:B] - gain[B:]
            if s["how"] == "sigmoid":
                good = torch.nn.functional.logsigmoid(BETA * m)
                bad = torch.nn.functional.logsigmoid(-BETA * m)
                loss = -(1 - s["smooth"]) * good - s["smooth"] * bad
            elif s["how"] == "hinge":
                loss = torch.relu(1 - BETA * m)
            else:
                loss = (m - 1 / (2 * BETA)) ** 2
            loss = loss.mean()
            c, = torch.autograd.grad(loss, total)
        out["loss"] = loss.detach()
        return torch.cat([c * unit, c.new_zeros(1)])[s["owner"]] * keep, None

    out["grad"] = _token_exact(s, tokens, make)[2].view(s["logits"].shape)
    return out
