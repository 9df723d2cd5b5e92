"""Beam search on the device: selection over beams and vocabulary, a whole decoding step, the
reordering of the beams' states and the answers (csrc/beam.hip, csrc/beam_states.hip; C ABI
``mvsd_beam_select``, ``mvsd_beam_step``, ``mvsd_beam_reorder``, ``mvsd_beam_finish``).

The reference has no beam search; this stands beside ``Sampler`` for requests that want the most
probable sequences.  A group is one request with W beams (1..64), G groups a batch, the rows of a
group's beams in the order g * W + w.

    search = BeamSearch(G, W, max_length, device, stop_token_ids=[eos])
    logits = prefill(...)                       # a row a beam (the first beam's counts)
    for _ in range(max_length):
        step = search.step(logits)              # step.token_ids, step.parents [G, W]
        search.reorder(caches, lengths=...)     # the beams' states follow their parents
        logits = decode(step.token_ids, caches)
    answers = search.finish(n)                  # token ids, lengths and scores of the n best

``search.state.done`` tells which groups are done, for a loop that ends earlier (reading it waits for the
device).  A group that reaches ``max_length`` rests with its flag unset: its running beams are answers.

Nothing here synchronises the host.  Work is enqueued on the current stream of the logits' (or
states') device.  Scratch is kept per stream; a captured call has its own, so calls on several
streams and captured graphs share nothing.
"""

from __future__ import annotations

import ctypes
import math
import struct
import threading
from dataclasses import dataclass

import torch

from .. import _native as nat

PLACEHOLDER_TOKEN_ID = -1
MAX_BEAMS = 64
MAX_CANDIDATES = 256

_ROW_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


@dataclass
class BeamCandidates:
    """The best continuations of every group, best first; [G, C] each.  Places without one:
    token and parent -1, score -inf."""

    token_ids: torch.Tensor  # int32
    parents: torch.Tensor    # int32, the beam (0..W-1) that each continues
    scores: torch.Tensor     # fp32, summed log-probabilities


@dataclass
class BeamState:
    """A search under way.  ``finished_*`` hold each group's W best finished hypotheses, best first
    (none: score -inf, -1, -1, 0): a hypothesis is its last token (``finished_token_ids``) appended
    to a beam (``finished_beams``) of the step before, ``finished_lengths`` tokens in all.
    ``token_history`` and ``parent_history`` hold what every step gave each beam."""

    scores: torch.Tensor              # fp32 [G, W], -inf: no beam
    lengths: torch.Tensor             # int32 [G], steps taken = tokens of the running beams
    done: torch.Tensor                # bool [G]; not set by reaching max_length
    finished_scores: torch.Tensor     # fp32 [G, W], divided by length ** length_penalty
    finished_beams: torch.Tensor      # int32 [G, W]
    finished_token_ids: torch.Tensor  # int32 [G, W]
    finished_lengths: torch.Tensor    # int32 [G, W]
    token_history: torch.Tensor       # int32 [G, max_length, W]
    parent_history: torch.Tensor      # int32 [G, max_length, W]

    @classmethod
    def new(cls, num_groups: int, beam_width: int, max_length: int, device) -> "BeamState":
        """Before the first step: beam 0 of every group holds the prompt."""
        G, W = num_groups, beam_width

        def full(value, dtype, *shape):
            return torch.full(shape, value, dtype=dtype, device=device)

        scores = full(-float("inf"), torch.float32, G, W)
        scores[:, 0] = 0.0
        return cls(scores, full(0, torch.int32, G), full(False, torch.bool, G),
                   full(-float("inf"), torch.float32, G, W), full(-1, torch.int32, G, W),
                   full(-1, torch.int32, G, W), full(0, torch.int32, G, W),
                   full(-1, torch.int32, G, max_length, W),
                   full(-1, torch.int32, G, max_length, W))


@dataclass
class BeamStep:
    """What the model runs next: [G, W] each, -1 where a group rests or has no such beam."""

    token_ids: torch.Tensor  # int32
    parents: torch.Tensor    # int32, the beam of the step before that each one continues
    state: BeamState


@dataclass
class BeamHypotheses:
    """The best answers of every group, best first."""

    token_ids: torch.Tensor  # int32 [G, n, max_length], -1 behind a sequence
    lengths: torch.Tensor    # int32 [G, n], 0: no such answer
    scores: torch.Tensor     # fp32 [G, n], -inf: no such answer


# A state's tensors in the order of mvsd_beam_step_args and mvsd_beam_finish_args: seven that a step
# replaces, then the histories.
_FIELDS = ("scores", "lengths", "done", "finished_scores", "finished_beams", "finished_token_ids",
           "finished_lengths")
_HISTORIES = ("token_history", "parent_history")
_I32, _F32 = torch.int32, torch.float32
_DTYPES = (_F32, _I32, torch.bool, _F32, _I32, _I32, _I32)
# the places of their addresses in the argument structures, in eight-byte words
_STEP_HEAD, _STEP_TENSORS = struct.Struct("=10qdii"), 12
_FINISH_HEAD, _FINISH_TENSORS = struct.Struct("=4qd"), 5
_STEP_TAIL, _FINISH_TAIL = struct.Struct("=4q"), struct.Struct("=5q")


_hostops = None


def _host():
    """The host extension, imported by the first call that needs it."""
    global _hostops
    if _hostops is None:
        from .. import _hostops as module

        _hostops = module
    return _hostops


def _check_array(t: torch.Tensor, name: str, dtype, shape, device) -> None:
    if t.dtype != dtype:
        raise TypeError(f"{name} is {t.dtype}, {dtype} expected")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, {tuple(shape)} expected")
    if t.device != device:
        nat.require_device_tensor(t, name)
        raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} is not contiguous")


def _addresses(args, at: int, names, tensors, dtypes, shapes, device) -> None:
    """The tensors' addresses into a call's arguments; raises for one of another kind."""
    bad = _host().tensor_table(args, at, tensors, dtypes, shapes, device)
    if bad >= 0:
        _check_array(tensors[bad], names[bad], dtypes[bad], shapes[bad], device)
        raise ValueError(f"{names[bad]} is no tensor that can be passed on")


def _fields(state: BeamState):
    return (state.scores, state.lengths, state.done, state.finished_scores, state.finished_beams,
            state.finished_token_ids, state.finished_lengths)


def _extent(state: BeamState) -> tuple[int, int, int]:
    history = state.token_history
    if history.ndim != 3:
        raise ValueError("token_history is not [G, max_length, W]")
    G, T, W = history.shape
    if not 1 <= W <= MAX_BEAMS:
        raise ValueError(f"{W} beams: 1 to {MAX_BEAMS} are supported")
    if T < 1:
        raise ValueError("the state has max_length 0")
    return G, T, W


def _elsewhere(device: torch.device) -> bool:
    """Whether `device` is not the current one, to which launches and allocations go."""
    return device.index is not None and device.index != torch.cuda.current_device()


def _check_rows(logits: torch.Tensor, G: int, W: int, target_rows) -> torch.device:
    nat.require_device_tensor(logits, "logits")
    if not 1 <= W <= MAX_BEAMS:
        raise ValueError(f"{W} beams: 1 to {MAX_BEAMS} are supported")
    if logits.ndim != 2 or logits.dtype not in _ROW_DTYPES:
        raise TypeError("logits are 2-D fp32, bf16 or fp16 rows")
    V = logits.shape[1]
    if V < 1:
        raise ValueError("logits without columns")
    if logits.stride(1) != 1 and V > 1:
        raise ValueError("logits need rows with unit stride")
    device = logits.device
    if target_rows is None:
        if logits.shape[0] < G * W:
            raise ValueError(f"{logits.shape[0]} logits rows for {G} groups of {W} beams")
    else:
        if target_rows.numel() != G * W:
            raise ValueError(f"{target_rows.numel()} row indices for {G} groups of {W} beams")
        _check_array(target_rows, "target_rows", torch.int32, target_rows.shape, device)
        if logits.shape[0] < 1 and G > 0:
            raise ValueError("row indices into logits without rows")
    return device


# Scratch of selections and steps, kept per (device, stream): calls on one stream follow each other.
# A call is two launches: _LOCK is held over both, so that two threads' do not mix on a stream.
_LOCK = threading.RLock()
_SCRATCH: dict[tuple[int, int], tuple[torch.Tensor, int, int]] = {}
_SCRATCH_MOST = 1 << 24


def _scratch(G: int, W: int, V: int, C: int, device: torch.device,
             stream: int) -> tuple[torch.Tensor, int, int]:
    """(workspace, its address, its size) of a call."""
    size = nat.lib().mvsd_beam_workspace_bytes(G, W, V, C)
    kept = _SCRATCH.get((device.index, stream))
    capturing = torch.cuda.is_current_stream_capturing()
    if kept is not None and kept[2] >= size > 0 and not capturing:
        return kept
    if size <= 0:
        raise ValueError(f"{G} groups of {W} beams over {V} tokens are more than one call takes")
    keep = size <= _SCRATCH_MOST and not capturing
    if keep and kept is not None:
        size = min(max(size, 2 * kept[2]), _SCRATCH_MOST)
    ws = torch.empty(size, dtype=torch.uint8, device=device)
    made = ws, ws.data_ptr(), size
    if keep:  # a captured call can be replayed beside later ones on this stream: it has its own
        _SCRATCH[device.index, stream] = made
    return made


def beam_search_select(logits: torch.Tensor, scores: torch.Tensor, num_candidates: int, *,
                       target_rows: torch.Tensor | None = None) -> BeamCandidates:
    """The ``num_candidates`` (1..256) best continuations of every group.

    ``scores [G, W]`` fp32 are the beams' summed log-probabilities, ``logits`` their rows (fp32,
    bf16 or fp16, any row stride): row g * W + w, or ``target_rows [G, W]`` (int32) into a larger
    tensor (indices outside it read its nearest row).  Candidate (beam, token) has the score
    ``scores[beam] + log_softmax(row)[token]``; the order, that of the 64-bit scores, is score
    descending, beam ascending, logit descending, token ascending (scores that differ in the last digits
    of 64-bit sums, as of a row and its permutation, may come either way).  The scores returned are
    formed in 64 bits from log-softmax values that are off by at most 2^-20, and by 2^-18 of themselves
    (fp32 exponentials), and rounded to fp32 (not past its lowest value).  A beam whose score is not finite, or whose row is -inf
    throughout or holds a NaN or +inf, proposes nothing; tokens at -inf are no candidates.
    """
    if scores.ndim != 2:
        raise ValueError("scores are [G, W]")
    G, W = scores.shape
    device = _check_rows(logits, G, W, target_rows)
    _check_array(scores, "scores", _F32, (G, W), device)
    C = int(num_candidates)
    if not 1 <= C <= MAX_CANDIDATES:
        raise ValueError(f"num_candidates={C}: 1 to {MAX_CANDIDATES} are supported")
    if _elsewhere(device):
        with torch.cuda.device(device):
            return beam_search_select(logits, scores, C, target_rows=target_rows)
    ids = torch.empty(3, G, C, dtype=_I32, device=device)
    token_ids, parents, bits = ids.unbind(0)
    out = BeamCandidates(token_ids, parents, bits.view(_F32))
    if G == 0:
        return out
    rows, V = logits.shape
    stream = nat.stream_of(device)
    base = ids.data_ptr()
    with _LOCK:
        scratch = _scratch(G, W, V, C, device, stream)
        status = nat.lib().mvsd_beam_select(
            base, base + 4 * G * C, base + 8 * G * C, logits.data_ptr(),
            nat.dtype_code(logits.dtype), logits.stride(0), rows, nat.ptr(target_rows),
            scores.data_ptr(), G, W, V, C, scratch[1], scratch[2], stream)
    nat.check(status, "mvsd_beam_select")
    return out


def beam_search_step(logits: torch.Tensor, state: BeamState, *,
                     stop_token_ids: torch.Tensor | None = None, length_penalty: float = 1.0,
                     early_stopping: bool = False, target_rows: torch.Tensor | None = None,
                     out: BeamState | None = None) -> BeamStep:
    """One decoding step of every group that is not done and has fewer than ``max_length`` tokens.

    With the candidates of :func:`beam_search_select` and L = length + 1:

    * stop tokens (``stop_token_ids``, int32 on the device, W * (1 + their number) <= 256) among the
      W best candidates end a hypothesis with score ``sum / L ** length_penalty`` (inside the range
      of fp32); each group keeps its W best, an earlier one first where they are equal;
    * the W best candidates that are no stop tokens are the next beams, also recorded in the
      histories;
    * the group is done when no beam is left, or when W hypotheses are finished and, unless
      ``early_stopping``, the worst of them is at least the best running sum / L ** length_penalty.

    Other groups stay as they are (token_ids and parents -1), also one that reached ``max_length`` and is
    not done: its running beams remain answers.  The new state is written to ``out``
    (another :class:`BeamState` with the same histories), or to ``state`` itself.
    """
    G, T, W = _extent(state)
    device = _check_rows(logits, G, W, target_rows)
    if out is None:
        out = state
    token_history, parent_history = state.token_history, state.parent_history
    if out is not state and (out.token_history is not token_history
                             or out.parent_history is not parent_history):
        if (out.token_history.data_ptr() != token_history.data_ptr()
                or out.parent_history.data_ptr() != parent_history.data_ptr()
                or out.token_history.shape != token_history.shape
                or out.parent_history.shape != parent_history.shape):
            raise ValueError("out has other histories than state")
    E = 0
    if stop_token_ids is not None:
        E = stop_token_ids.numel()
        _check_array(stop_token_ids, "stop_token_ids", _I32, (E,), device)
    C = W * (1 + E)
    if C > MAX_CANDIDATES:
        raise ValueError(f"{W} beams with {E} stop tokens: W * (1 + E) is over {MAX_CANDIDATES}")
    if _elsewhere(device):
        with torch.cuda.device(device):
            return beam_search_step(logits, state, stop_token_ids=stop_token_ids,
                                    length_penalty=length_penalty, early_stopping=early_stopping,
                                    target_rows=target_rows, out=out)
    if not math.isfinite(length_penalty):
        raise ValueError(f"length_penalty={length_penalty}")
    args = nat.BeamStepArgs()
    a, b, c = (G, W), (G,), (G, T, W)
    fields = (a, b, b, a, a, a, a)
    old, new = _fields(state), _fields(out)
    _addresses(args, _STEP_TENSORS, _STEP_NAMES, old + new + (token_history, parent_history),
               _STEP_DTYPES, fields + fields + (c, c), device)
    token_ids = torch.empty_like(state.finished_beams)
    parents = torch.empty_like(state.finished_beams)
    step = BeamStep(token_ids, parents, out)
    if G == 0:
        return step
    rows, V = logits.shape
    stream = nat.stream_of(device)
    _STEP_HEAD.pack_into(args, 0, logits.data_ptr(), logits.stride(0), rows,
                         0 if target_rows is None else target_rows.data_ptr(), G, W, V, T,
                         stop_token_ids.data_ptr() if E else 0, E, length_penalty,
                         nat.dtype_code(logits.dtype), 1 if early_stopping else 0)
    with _LOCK:
        scratch = _scratch(G, W, V, C, device, stream)
        _STEP_TAIL.pack_into(args, 8 * (_STEP_TENSORS + 16), token_ids.data_ptr(),
                             parents.data_ptr(), scratch[1], scratch[2])
        status = nat.lib().mvsd_beam_step(ctypes.byref(args), stream)
    nat.check(status, "mvsd_beam_step")
    return step


_STEP_NAMES = tuple("state." + f for f in _FIELDS) + tuple("out." + f for f in _FIELDS) \
    + tuple("state." + f for f in _HISTORIES)
_STEP_DTYPES = _DTYPES + _DTYPES + (_I32, _I32)
_FINISH_NAMES = tuple("state." + f for f in _FIELDS + _HISTORIES)
_FINISH_DTYPES = _DTYPES + (_I32, _I32)


def beam_search_finish(state: BeamState, num_return: int | None = None, *,
                       length_penalty: float = 1.0) -> BeamHypotheses:
    """The ``num_return`` (default W) best answers of every group: its finished hypotheses and, unless
    the group is done, its running beams (sum / length ** length_penalty); finished ones first where
    they are equal.  The sequences are read back from the histories; the state is left as it is."""
    nat.require_device_tensor(state.scores, "state.scores")
    device = state.scores.device
    G, T, W = _extent(state)
    n = W if num_return is None else int(num_return)
    if not 1 <= n <= W:
        raise ValueError(f"num_return={n}: 1 to {W} (the beams) are kept")
    if _elsewhere(device):
        with torch.cuda.device(device):
            return beam_search_finish(state, n, length_penalty=length_penalty)
    if not math.isfinite(length_penalty):
        raise ValueError(f"length_penalty={length_penalty}")
    args = nat.BeamFinishArgs()
    a, b, c = (G, W), (G,), (G, T, W)
    _addresses(args, _FINISH_TENSORS, _FINISH_NAMES,
               _fields(state) + (state.token_history, state.parent_history), _FINISH_DTYPES,
               (a, b, b, a, a, a, a, c, c), device)
    ids = torch.empty(G, n, T, dtype=_I32, device=device)
    lengths = torch.empty(G, n, dtype=_I32, device=device)
    scores = torch.empty(G, n, dtype=_F32, device=device)
    out = BeamHypotheses(ids, lengths, scores)
    if G == 0:
        return out
    size = nat.lib().mvsd_beam_finish_workspace_bytes(G, W, T, n)
    ws = torch.empty(size, dtype=torch.uint8, device=device) if size > 0 else None
    _FINISH_HEAD.pack_into(args, 0, G, W, T, n, length_penalty)
    _FINISH_TAIL.pack_into(args, 8 * (_FINISH_TENSORS + 9), ids.data_ptr(), lengths.data_ptr(),
                           scores.data_ptr(), 0 if ws is None else ws.data_ptr(), size)
    nat.check(nat.lib().mvsd_beam_finish(ctypes.byref(args), nat.stream_of(device)),
              "mvsd_beam_finish")
    return out


def _refuse_states(tensors, targets, length_dim: int, device, least_rows: int) -> None:
    """Raises for the first of the tensors that is no state."""
    for k, (x, to) in enumerate(zip(tensors, targets)):
        for t, name in ((x, f"states[{k}]"), (to, f"out[{k}]")):
            nat.require_device_tensor(t, name)
            if t.device != device:
                raise ValueError(f"{name} is on {t.device}, parents on {device}")
            if not 1 <= length_dim < t.ndim:
                raise ValueError(f"{name} has no dimension {length_dim} behind its rows")
            if t.shape[0] < least_rows:
                raise ValueError(f"{name} has {t.shape[0]} rows for {least_rows} beams")
            if t.shape != x.shape or t.dtype != x.dtype:
                raise ValueError(f"{name} has another shape or dtype than states[{k}]")
            if t.numel() and not t[0].is_contiguous():
                raise ValueError(f"{name} is not contiguous within a row")
            if t.shape[0] > 1 and t.numel() and t.stride(0) < t[0].numel():
                raise ValueError(f"{name} has overlapping rows")
    raise ValueError("a state is no tensor that can be passed on")


def _reorder_refusal(table, n: int) -> str:
    """Why mvsd_beam_reorder refuses states that _hostops.state_table took."""
    same = [table[8 * k] == table[8 * k + 1] for k in range(n)]
    if any(same) and not all(same):
        return "out names some of the states: all are reordered in place or none"
    if any(s and table[8 * k + 2] != table[8 * k + 3] for k, s in enumerate(same)):
        return "out has a state's memory with another row stride"
    return "the states (or out) share memory with each other"


def reorder_beams(states, parents: torch.Tensor, *, starts: torch.Tensor | None = None,
                  lengths: torch.Tensor | None = None, length_dim: int = 1,
                  slots: torch.Tensor | None = None, out=None):
    """The states of the beams follow their parents: the row of beam (g, w) becomes what the row of
    beam (g, ``parents[g, w]``) was before the call.

    ``states`` is a tensor or a sequence of tensors (caches, token tables; any dtype), one row a
    beam along dimension 0 -- row g * W + w, or ``slots [G, W]`` (int32, distinct) into a pool of
    rows -- contiguous within a row, any row stride.  ``length_dim`` is the dimension of the
    positions in all of them; only positions ``starts[g] <= t < lengths[g]`` (int32 [G]; default:
    all) move, so a prompt that the beams of a group share can stay where it is.  A parent outside
    0..W-1 (the -1 of a resting group) keeps the beam's own row; a slot outside the pool is left
    alone.

    At most 512 tensors a call, rows below 16 GiB, no memory in common except rows that interleave
    with equal strides (keys and values of one tensor).

    Without ``out`` the states are reordered in place, in one pass and without a second buffer; with
    ``out`` (tensors of the same shapes that share no memory with the states) the rows are written
    there.  Returns the tensors written.  Nothing else is touched.
    """
    if parents.ndim != 2:
        raise ValueError("parents are [G, W]")
    nat.require_device_tensor(parents, "parents")
    device = parents.device
    G, W = parents.shape
    if not 1 <= W <= MAX_BEAMS:
        raise ValueError(f"{W} beams: 1 to {MAX_BEAMS} are supported")
    _check_array(parents, "parents", torch.int32, (G, W), device)
    if starts is not None:
        _check_array(starts, "starts", torch.int32, (G,), device)
    if lengths is not None:
        _check_array(lengths, "lengths", torch.int32, (G,), device)
    if slots is not None:
        _check_array(slots, "slots", torch.int32, (G, W), device)
    single = isinstance(states, torch.Tensor)
    tensors = (states,) if single else tuple(states)
    targets = tensors if out is None else (out,) if isinstance(out, torch.Tensor) else tuple(out)
    if len(targets) != len(tensors):
        raise ValueError(f"{len(targets)} out tensors for {len(tensors)} states")
    table = (ctypes.c_int64 * (8 * len(tensors)))()
    n = _host().state_table(table, tensors, targets, length_dim, device,
                            0 if slots is not None else G * W)
    if n < 0:
        _refuse_states(tensors, targets, length_dim, device, 0 if slots is not None else G * W)
    if n and G:
        call = (table, n, parents.data_ptr(), nat.ptr(starts), nat.ptr(lengths), nat.ptr(slots),
                G, W, nat.stream_of(device))
        if _elsewhere(device):
            with torch.cuda.device(device):
                status = nat.lib().mvsd_beam_reorder(*call)
        else:
            status = nat.lib().mvsd_beam_reorder(*call)
        if status == -1:
            raise ValueError(_reorder_refusal(table, n))
        nat.check(status, "mvsd_beam_reorder")
    return targets[0] if single else list(targets)


class BeamSearch:
    """A beam search of G requests: its state, step by step (see the module's example)."""

    def __init__(self, num_groups: int, beam_width: int, max_length: int, device, *,
                 stop_token_ids=(), length_penalty: float = 1.0, early_stopping: bool = False):
        if not 1 <= beam_width <= MAX_BEAMS:
            raise ValueError(f"{beam_width} beams: 1 to {MAX_BEAMS} are supported")
        if max_length < 1:
            raise ValueError("max_length is at least 1")
        if beam_width * (1 + len(stop_token_ids)) > MAX_CANDIDATES:
            raise ValueError(f"{beam_width} beams with {len(stop_token_ids)} stop tokens: "
                             f"W * (1 + E) is over {MAX_CANDIDATES}")
        self.state = BeamState.new(num_groups, beam_width, max_length, device)
        self.stop_token_ids = torch.tensor(list(stop_token_ids), dtype=torch.int32, device=device)
        self.length_penalty = float(length_penalty)
        self.early_stopping = bool(early_stopping)
        self.parents: torch.Tensor | None = None

    def step(self, logits: torch.Tensor, target_rows: torch.Tensor | None = None) -> BeamStep:
        """One step on the beams' logits (:func:`beam_search_step`); the state is updated."""
        step = beam_search_step(logits, self.state, stop_token_ids=self.stop_token_ids,
                                length_penalty=self.length_penalty,
                                early_stopping=self.early_stopping, target_rows=target_rows)
        self.parents = step.parents
        return step

    def reorder(self, states, **where):
        """The states of the beams follow the last step's parents (:func:`reorder_beams`)."""
        if self.parents is None:
            raise RuntimeError("no step has been taken")
        return reorder_beams(states, self.parents, **where)

    def finish(self, num_return: int | None = None) -> BeamHypotheses:
        """The best answers so far (:func:`beam_search_finish`)."""
        return beam_search_finish(self.state, num_return, length_penalty=self.length_penalty)
