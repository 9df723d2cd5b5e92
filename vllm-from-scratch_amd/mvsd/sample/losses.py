"""Training losses on rows of logits, with their gradients (csrc/losses.hip; C ABI ``mvsd_row_loss``,
``mvsd_loss_gradient``): what is learnt from the tokens, log-probabilities and answers that the
samplers, the verification and beam search give.  The reference has none of them.

* :func:`token_logprobs`: log-probabilities (and entropies) of given tokens;
* :func:`distillation_loss`: a draft model against the target's top log-probabilities, as
  ``compute_topk_scores`` and the speculative logprobs return them;
* :func:`policy_loss`: clipped policy loss with a KL term and an entropy bonus;
* :func:`preference_loss`: paired log ratios of whole answers.

    scores = compute_topk_scores(target_logits, 32, sampled)       # while serving
    loss = distillation_loss(draft_logits, scores.logprob_token_ids, scores.logprobs)
    loss.backward()

``logits`` are [N, V] or [B, L, V] in fp32, bf16 or fp16, any strides over the rows, unit stride within
one.  Values of a row have the leading shape, fp32; what has fewer dimensions or ones is expanded.  Token
ids are int32 or int64.  A row whose id is negative (distillation: that has no entry) or whose weight is
0 is left out: its logits are not read, its values and its gradient are 0.  An id of V or more, or a row
with a NaN, a +inf or nothing but -inf in it, gives NaN.  The logits get gradients, once differentiable
and not in forward mode, in their own dtype; every other argument is a constant.  Values and losses are fp32.

Reductions: "mean" is sum(w * l) / sum(w) over the rows that are not left out (0 if there are none),
"sum" is sum(w * l), so weights carry any other normalisation and loss scales, "none" the w * l.

A policy or distillation loss that is a scalar over many rows forms the logits' gradient for an upstream
of 1 in the forward pass, where it reads them, and saves it for the backward pass (a kept graph holds it);
for another upstream the rows are read again, for 2.2 to 2.6 times the time of both passes (a scale in
``weights`` with "sum" avoids that).  Leave rows out by their ids
instead of indexing the logits, which copies them.

Nothing here synchronises the host; work is enqueued on the current stream of the logits' device and may
be captured into a graph.  Before a backward pass is captured, release graphs of the same leaves that ran
eagerly (torch ends the process otherwise).
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import torch
from torch.autograd import forward_ad

from .. import _native as nat

MAX_TEACHER_TOKENS = 512
_SMALL_SCRATCH = 1 << 18

_ROW_CODES = {t: nat.dtype_code(t) for t in (torch.float32, torch.bfloat16, torch.float16)}
_ID_CODES = {t: nat.dtype_code(t) for t in (torch.int32, torch.int64)}
_LOGPROBS, _DISTILL, _POLICY, _PREFERENCE = range(4)
_REDUCTIONS = {"sum": 0, "mean": 1, "none": 2}
_DIVERGENCES = {"forward": 0, "reverse": 1, "js": 2}
_LOSS_TYPES = {"sigmoid": 0, "hinge": 1, "squared": 2}


@dataclass
class PolicyLoss:
    """``loss`` is differentiable; the rows' values are not."""

    loss: torch.Tensor
    logprobs: torch.Tensor        # of the tokens
    entropy: torch.Tensor | None  # with an entropy coefficient
    kl: torch.Tensor | None       # e^d - d - 1, d = ref - lp, with reference log-probabilities


@dataclass
class PreferenceLoss:
    """``loss`` is differentiable; the sequences' values are not."""

    loss: torch.Tensor
    logprobs: torch.Tensor  # [2 * pairs], the chosen then the rejected sequences'


def _choice(value, choices: dict, name: str) -> int:
    try:
        return choices[value]
    except (KeyError, TypeError):
        raise ValueError(f"{name}={value!r}: one of {', '.join(choices)}") from None


def _number(value, name: str) -> float:
    value = float(value)
    if not math.isfinite(value):
        raise ValueError(f"{name}={value}")
    return value


def _check_device(t: torch.Tensor, name: str, device: torch.device) -> None:
    nat.require_device_tensor(t, name)
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the logits on {device}")


def _check_ids(ids: torch.Tensor, name: str, shape, device) -> torch.Tensor:
    if ids.dtype in _ID_CODES and ids.shape == shape and ids.device == device:
        return ids if ids.is_contiguous() else ids.contiguous()
    _check_device(ids, name, device)
    if ids.dtype not in _ID_CODES:
        raise TypeError(f"{name} is {ids.dtype}, int32 or int64 expected")
    raise ValueError(f"{name} has shape {tuple(ids.shape)}, {tuple(shape)} expected")


def _values(t: torch.Tensor, name: str, shape, device) -> torch.Tensor:
    """An fp32 value for every place of `shape`."""
    if t.dtype is torch.float32 and t.shape == shape and t.device == device and t.is_contiguous():
        return t
    _check_device(t, name, device)
    if t.dtype != torch.float32:
        raise TypeError(f"{name} is {t.dtype}, torch.float32 expected")
    if t.shape != shape:
        try:
            t = t.detach().expand(shape)
        except RuntimeError:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, {tuple(shape)} expected") from None
    return t.detach().contiguous()


class _Call:
    """One call: its arguments and the tensors they point to."""

    __slots__ = ("args", "kind", "logits", "ids", "keep", "outputs", "saved", "grad", "fresh",
                 "device", "layout")

    def __init__(self, kind: int, logits: torch.Tensor, temperature: float, reduction: int):
        if not logits.is_cuda:
            nat.require_device_tensor(logits, "logits")
        if logits.ndim not in (2, 3) or logits.dtype not in _ROW_CODES:
            raise TypeError("logits are [N, V] or [B, L, V] in fp32, bf16 or fp16")
        if logits.shape[-1] < 1:
            raise ValueError("logits without columns")
        temperature = float(temperature)
        if not 1e-6 <= temperature <= 1e6:
            raise ValueError(f"temperature={temperature}")
        self.kind, self.logits, self.device = kind, logits, logits.device
        self.keep, self.saved, self.grad, self.fresh = [], None, None, [True]
        a = self.args = nat.LossArgs()
        a.kind, a.reduction, a.temperature = kind, reduction, temperature
        self.layout = self._rows(a, logits)

    @staticmethod
    def _rows(a: nat.LossArgs, logits: torch.Tensor) -> tuple:
        shape, strides, data = logits.shape, logits.stride(), logits.data_ptr()
        if strides[-1] != 1 and shape[-1] > 1:
            raise ValueError("logits need rows with unit stride")
        a.dtype = _ROW_CODES[logits.dtype]
        a.logits, a.vocab_size, a.stride = data, shape[-1], strides[-2]
        if len(shape) == 3:
            a.num_rows = shape[0] * shape[1]
            a.inner_rows, a.outer_stride = max(shape[1], 1), strides[0]
        else:
            a.num_rows = shape[0]
            a.inner_rows, a.outer_stride = max(shape[0], 1), 0
        return data, strides

    def take_ids(self, ids: torch.Tensor) -> None:
        self.ids = ids
        self.args.token_ids, self.args.ids_dtype = ids.data_ptr(), _ID_CODES[ids.dtype]

    def take(self, name: str, t: torch.Tensor | None, shape) -> None:
        if t is not None:
            t = _values(t, name, shape, self.device)
            self.keep.append(t)
            setattr(self.args, name, t.data_ptr())

    def take_weights(self, t: torch.Tensor | None, shape) -> None:
        if t is not None:
            self.take("weights", t.to(torch.float32) if t.dtype is torch.bool else t, shape)

    def empty(self, name: str, shape) -> torch.Tensor:
        out = torch.empty(shape, dtype=torch.float32, device=self.device)
        setattr(self.args, name, out.data_ptr())
        return out

    def run(self, train: bool) -> None:
        """Enqueue the values, and what the gradient needs of them."""
        a, handle = self.args, nat.lib()
        ref = ctypes.byref(a)
        if handle.mvsd_loss_plan(ref) != 0:
            raise ValueError(f"logits {tuple(self.logits.shape)} are more than one call takes")
        device, scratch = self.device, a.workspace_bytes
        if train:
            # what is saved, with a small call's scratch behind it
            kept = (a.saved_bytes + 15) // 16 * 16
            with_it = scratch <= _SMALL_SCRATCH
            self.saved = torch.empty(kept + scratch if with_it else kept, dtype=torch.uint8, device=device)
            a.saved = self.saved.data_ptr() or None
            if a.one_pass:
                self.grad = torch.empty(self.logits.shape, dtype=self.logits.dtype, device=device)
                a.grad = self.grad.data_ptr()
            if with_it:
                a.workspace = (a.saved or 0) + kept
        if not a.workspace:
            workspace = torch.empty(scratch, dtype=torch.uint8, device=device)
            a.workspace = workspace.data_ptr()
        status = handle.mvsd_row_loss(ref, nat.stream_of(device))
        if status != 0:
            nat.check(status, "mvsd_row_loss")
        self.keep = None

    def gradient(self, logits, ids, saved, unit, upstream, upstream_entropy) -> torch.Tensor:
        """The logits' gradient for the outputs' (a tensor may lie elsewhere than when it was saved);
        ``unit``: that of an upstream of 1, where it is there already, or None."""
        # several threads may go back through a kept graph at once: a pass's own arguments
        a = nat.LossArgs.from_buffer_copy(self.args)
        if self.layout != (logits.data_ptr(), logits.stride()):
            self._rows(a, logits)
        a.token_ids, a.saved = ids.data_ptr(), saved.data_ptr() or None
        # it goes out once, free to be changed (an alias without its version): a kept graph's next is made anew
        try:
            fresh = unit is not None and self.fresh.pop()
        except IndexError:
            fresh = False
        a.unit_gradient = 1 if fresh else 0
        grad = unit.data if fresh else torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        if grad.numel() == 0:
            return grad
        a.grad = grad.data_ptr()
        ups, kept = [], []
        for g in (upstream, upstream_entropy):
            if g is None:
                ups += (None, 0)
                continue
            if g.dtype is not torch.float32 or not g.is_contiguous():
                g = g.to(torch.float32).contiguous()
                kept.append(g)
            ups += (g.data_ptr(), 1 if g.ndim else 0)
        status = nat.lib().mvsd_loss_gradient(ctypes.byref(a), *ups, nat.stream_of(logits.device))
        if status != 0:
            nat.check(status, "mvsd_loss_gradient")
        return grad


def _backward(ctx, upstream, *others):
    logits, ids, saved, *unit = ctx.saved_tensors
    call, unit = ctx.call, unit[0] if unit else None
    entropy = others[0] if call.kind == _LOGPROBS and others else None
    if upstream is None and entropy is None:
        return None, None
    if logits.device.index == torch.cuda.current_device():
        return call.gradient(logits, ids, saved, unit, upstream, entropy), None
    with torch.cuda.device(logits.device):
        return call.gradient(logits, ids, saved, unit, upstream, entropy), None


class _RowLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, call):
        call.run(True)
        ctx.set_materialize_grads(False)
        if call.kind != _LOGPROBS and len(call.outputs) > 1:
            ctx.mark_non_differentiable(*call.outputs[1:])
        # the gradient that is there already among them, so that hooks and recomputation see it
        if call.grad is None:
            ctx.save_for_backward(logits, call.ids, call.saved)
        else:
            ctx.save_for_backward(logits, call.ids, call.saved, call.grad)
        outputs, call.outputs = call.outputs, ()
        call.logits = call.ids = call.saved = call.grad = None
        ctx.call = call
        return outputs

    @staticmethod
    def backward(ctx, *upstream):
        if torch.is_grad_enabled():  # a graph of the gradient is asked for, which there is not
            return _refusing_backward(ctx, *upstream)
        return _backward(ctx, *upstream)


_refusing_backward = torch.autograd.function.once_differentiable(_backward)


def _finish(call: _Call):
    """The call's outputs, part of the graph where the logits want a gradient."""
    if forward_ad.unpack_dual(call.logits).tangent is not None:
        raise NotImplementedError("the losses have no forward-mode derivatives: detach the logits")
    if call.logits.requires_grad and torch.is_grad_enabled():
        return _RowLoss.apply(call.logits, call)
    call.run(False)
    return call.outputs


def _on_device(logits) -> bool:
    """Whether the logits' device is the current one, to which launches and allocations go."""
    return not logits.is_cuda or logits.device.index == torch.cuda.current_device()


def token_logprobs(logits: torch.Tensor, token_ids: torch.Tensor, *, temperature: float = 1.0,
                   return_entropy: bool = False):
    """``log_softmax(logits / temperature)`` at ``token_ids``, in the leading shape; with
    ``return_entropy`` also the rows' entropies, both differentiable.

    A token's log-probability is formed from its odds against all others, so that one close to 0 keeps
    its digits."""
    if not _on_device(logits):
        with torch.cuda.device(logits.device):
            return token_logprobs(logits, token_ids, temperature=temperature,
                                  return_entropy=return_entropy)
    call = _Call(_LOGPROBS, logits, temperature, 0)
    lead = logits.shape[:-1]
    call.take_ids(_check_ids(token_ids, "token_ids", lead, call.device))
    call.outputs = (call.empty("logprobs", lead),)
    if return_entropy:
        call.outputs += (call.empty("entropy", lead),)
    out = _finish(call)
    return out if return_entropy else out[0]


def distillation_loss(logits: torch.Tensor, teacher_token_ids: torch.Tensor,
                      teacher_logprobs: torch.Tensor, *, divergence: str = "forward",
                      tail: bool = True, temperature: float = 1.0,
                      weights: torch.Tensor | None = None, reduction: str = "mean") -> torch.Tensor:
    """The divergence between a teacher's top tokens and ``p = softmax(logits / temperature)``.

    ``teacher_token_ids`` and ``teacher_logprobs`` (fp32) are [..., K], K up to 512.  Negative ids are
    no entries; a token that stands in a row twice counts at its first place (the sampled token in
    front of its row's top ones).

    * With ``tail``, the outcomes are the entries and, as one, the rest of the vocabulary:
      ``q = exp(teacher_logprobs)``, and for the rest 1 minus their sum (at least 2^-24, about what
      fp32 log-probabilities resolve; if the entries are the whole vocabulary there is no rest).  The
      teacher's log-probabilities are taken as they are, at the teacher's temperature.
    * Without, ``q = softmax(teacher_logprobs / temperature)`` over the entries alone (logits do as
      well); "forward" only.

    ``divergence``: "forward" is KL(q | p), "reverse" KL(p | q), "js" the mean of both against
    (p + q) / 2.  A p below fp32's range is 0: it adds nothing to "reverse", also where q is 0.
    """
    if not _on_device(logits):
        with torch.cuda.device(logits.device):
            return distillation_loss(logits, teacher_token_ids, teacher_logprobs,
                                     divergence=divergence, tail=tail, temperature=temperature,
                                     weights=weights, reduction=reduction)
    call = _Call(_DISTILL, logits, temperature, _choice(reduction, _REDUCTIONS, "reduction"))
    a, lead = call.args, logits.shape[:-1]
    a.divergence, a.tail = _choice(divergence, _DIVERGENCES, "divergence"), 1 if tail else 0
    if divergence != "forward" and not tail:
        raise ValueError(f'divergence="{divergence}" needs the tail')
    if teacher_token_ids.ndim != logits.ndim:
        raise ValueError("teacher_token_ids are the logits' leading shape and K entries")
    K = a.num_teacher = teacher_token_ids.shape[-1]
    if not 1 <= K <= MAX_TEACHER_TOKENS:
        raise ValueError(f"{K} teacher tokens: 1 to {MAX_TEACHER_TOKENS} are supported")
    call.take_ids(_check_ids(teacher_token_ids, "teacher_token_ids", lead + (K,), call.device))
    call.take("teacher_logprobs", teacher_logprobs, lead + (K,))
    call.take_weights(weights, lead)
    call.outputs = (call.empty("loss", lead if reduction == "none" else ()),)
    return _finish(call)[0]


def policy_loss(logits: torch.Tensor, token_ids: torch.Tensor, old_logprobs: torch.Tensor | None,
                advantages: torch.Tensor, *, ref_logprobs: torch.Tensor | None = None,
                clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0,
                entropy_coef: float = 0.0, temperature: float = 1.0,
                weights: torch.Tensor | None = None, reduction: str = "mean") -> PolicyLoss:
    """Clipped policy loss of sampled tokens: with lp their log-probabilities under
    ``softmax(logits / temperature)`` and r = exp(lp - old_logprobs),

        l = -min(r * A, clip(r, 1 - clip_low, 1 + clip_high) * A)
            + kl_coef * (exp(d) - d - 1) - entropy_coef * H,    d = ref_logprobs - lp

    ``old_logprobs`` None stands for lp itself (r = 1, with lp's gradient); without ``ref_logprobs``
    there is no KL term.  At a border of the clip the gradient is the unclipped one."""
    if not _on_device(logits):
        with torch.cuda.device(logits.device):
            return policy_loss(logits, token_ids, old_logprobs, advantages,
                               ref_logprobs=ref_logprobs, clip_low=clip_low, clip_high=clip_high,
                               kl_coef=kl_coef, entropy_coef=entropy_coef, temperature=temperature,
                               weights=weights, reduction=reduction)
    call = _Call(_POLICY, logits, temperature, _choice(reduction, _REDUCTIONS, "reduction"))
    a, lead = call.args, logits.shape[:-1]
    a.clip_low, a.clip_high = _number(clip_low, "clip_low"), _number(clip_high, "clip_high")
    if a.clip_low < 0 or a.clip_high < 0:
        raise ValueError(f"clip_low={clip_low}, clip_high={clip_high}")
    a.kl_coef, a.entropy_coef = _number(kl_coef, "kl_coef"), _number(entropy_coef, "entropy_coef")
    if a.kl_coef != 0 and ref_logprobs is None:
        raise ValueError("kl_coef without ref_logprobs")
    call.take_ids(_check_ids(token_ids, "token_ids", lead, call.device))
    if advantages is None:
        raise ValueError("advantages are needed")
    call.take("advantages", advantages, lead)
    call.take("old_logprobs", old_logprobs, lead)
    call.take("ref_logprobs", ref_logprobs, lead)
    call.take_weights(weights, lead)
    outputs = [call.empty("loss", lead if reduction == "none" else ()),
               call.empty("logprobs", lead)]
    if a.entropy_coef != 0:
        outputs.append(call.empty("entropy", lead))
    if ref_logprobs is not None:
        outputs.append(call.empty("kl", lead))
    call.outputs = tuple(outputs)
    with_entropy = a.entropy_coef != 0
    loss, logprobs, *rest = _finish(call)
    return PolicyLoss(loss, logprobs, rest.pop(0) if with_entropy else None,
                      rest.pop(0) if rest else None)


def preference_loss(logits: torch.Tensor, token_ids: torch.Tensor,
                    ref_logprobs: torch.Tensor | None = None, *,
                    cu_num_tokens: torch.Tensor | None = None, beta: float = 0.1,
                    loss_type: str = "sigmoid", label_smoothing: float = 0.0, margin: float = 0.0,
                    average: bool = False, temperature: float = 1.0,
                    weights: torch.Tensor | None = None, reduction: str = "mean") -> PreferenceLoss:
    """A loss on pairs of answers: sequences 0..B-1 are the chosen ones, B..2B-1 the rejected ones.

    The sequences are the rows of ``logits [2B, L, V]`` (padding and prompts: token -1), or lie one
    behind the other in ``logits [N, V]``: sequence s is rows ``cu_num_tokens[s - 1]`` to
    ``cu_num_tokens[s]`` (int32 [2B], inclusive sums without a leading 0, never decreasing; rows behind
    the last one belong to none).  With S a sequence's summed log-probability (``average``: over the
    number of its tokens; an empty one has 0), m = (S - ref)_chosen - (S - ref)_rejected and
    h = beta * m - margin:

    * "sigmoid": -(1 - label_smoothing) * log sigmoid(h) - label_smoothing * log sigmoid(-h);
    * "hinge": max(0, 1 - h);
    * "squared": (m - margin - 1 / (2 * beta)) ** 2.

    ``ref_logprobs`` fp32 [2B] are the reference model's S (None: 0); ``weights`` [B] the pairs'."""
    if not _on_device(logits):
        with torch.cuda.device(logits.device):
            return preference_loss(logits, token_ids, ref_logprobs, cu_num_tokens=cu_num_tokens,
                                   beta=beta, loss_type=loss_type, label_smoothing=label_smoothing,
                                   margin=margin, average=average, temperature=temperature,
                                   weights=weights, reduction=reduction)
    call = _Call(_PREFERENCE, logits, temperature, _choice(reduction, _REDUCTIONS, "reduction"))
    a, lead = call.args, logits.shape[:-1]
    a.loss_type, a.average = _choice(loss_type, _LOSS_TYPES, "loss_type"), 1 if average else 0
    a.beta, a.margin = _number(beta, "beta"), _number(margin, "margin")
    a.label_smoothing = _number(label_smoothing, "label_smoothing")
    if a.beta <= 0:
        raise ValueError(f"beta={beta}")
    if not 0 <= a.label_smoothing <= 1 or (a.label_smoothing and loss_type != "sigmoid"):
        raise ValueError(f'label_smoothing={label_smoothing} with loss_type="{loss_type}"')
    if (cu_num_tokens is None) != (logits.ndim == 3):
        raise ValueError("logits [2B, L, V], or [N, V] with cu_num_tokens")
    if cu_num_tokens is not None:
        _check_device(cu_num_tokens, "cu_num_tokens", call.device)
        if cu_num_tokens.dtype != torch.int32 or cu_num_tokens.ndim != 1:
            raise TypeError("cu_num_tokens is int32 [2B]")
        sequences = cu_num_tokens.shape[0]
        call.keep.append(cu_num_tokens.contiguous())
        a.cu_num_tokens = call.keep[0].data_ptr()
    else:
        sequences = lead[0]
    if sequences % 2:
        raise ValueError(f"{sequences} sequences are no pairs")
    B = a.num_pairs = sequences // 2
    call.take_ids(_check_ids(token_ids, "token_ids", lead, call.device))
    call.take("ref_logprobs", ref_logprobs, (2 * B,))
    call.take_weights(weights, (B,))
    call.outputs = (call.empty("loss", (B,) if reduction == "none" else ()),
                    call.empty("logprobs", (2 * B,)))
    return PreferenceLoss(*_finish(call))
