"""Beam search without a GPU: the C ABI's refusals and struct layouts, the Python layer's refusals."""

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from mvsd import _hostops
from mvsd import _native as nat
from mvsd.sample import (BeamSearch, BeamState, beam_search_finish, beam_search_select,
                         beam_search_step, reorder_beams)

HEADER = Path(__file__).resolve().parents[1] / "include" / "mvsd.h"
INVALID, WORKSPACE, RANGE = -1, -3, -5


@pytest.mark.parametrize("name,fields", [
    ("mvsd_beam_step_args", [(f, getattr(nat.BeamStepArgs, f).offset)
                             for f, _ in nat.BeamStepArgs._fields_]),
    ("mvsd_beam_finish_args", [(f, getattr(nat.BeamFinishArgs, f).offset)
                               for f, _ in nat.BeamFinishArgs._fields_]),
    ("mvsd_beam_state", [(f, 8 * i) for i, f in enumerate(
        ("src", "dst", "src_stride", "dst_stride", "num_rows", "outer", "length", "inner"))])])
def test_struct_layouts(tmp_path, name, fields):
    size = {"mvsd_beam_step_args": ctypes.sizeof(nat.BeamStepArgs),
            "mvsd_beam_finish_args": ctypes.sizeof(nat.BeamFinishArgs), "mvsd_beam_state": 64}[name]
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){",
             f'printf("%zu\\n", sizeof({name}));']
    lines += [f'printf("%zu\\n", offsetof({name}, {f}));' for f, _ in fields] + ["return 0;}"]
    (tmp_path / "probe.c").write_text("\n".join(lines))
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-o", str(exe), str(tmp_path / "probe.c")], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    assert got == [size] + [at for _, at in fields]


def test_workspace_sizes():
    size = nat.lib().mvsd_beam_workspace_bytes
    assert 0 < size(1, 4, 151936, 8) < size(64, 4, 151936, 8)
    for bad in [(1, 0, 10, 1), (1, 65, 10, 1), (1, 4, 0, 1), (1, 4, 10, 0), (1, 4, 10, 257),
                (-1, 4, 10, 1), (1, 4, 2 ** 31, 1), (2 ** 25, 64, 10, 1), (2 ** 20, 64, 10, 1)]:
        assert size(*bad) == 0, bad


P = 1 << 20  # an address that no refused call touches


def select(token_ids=P, parents=P, scores=P, logits=P, dtype=0, stride=100, rows=8, target=None,
           beam_scores=P, G=2, W=4, V=100, C=8, ws=P, ws_bytes=1 << 20):
    return nat.lib().mvsd_beam_select(token_ids, parents, scores, logits, dtype, stride, rows,
                                      target, beam_scores, G, W, V, C, ws, ws_bytes, None)


@pytest.mark.parametrize("change,status", [
    ({"W": 0}, INVALID), ({"W": 65}, RANGE), ({"C": 0}, INVALID), ({"C": 257}, RANGE),
    ({"G": -1}, INVALID), ({"G": 2 ** 40}, RANGE), ({"V": 0}, INVALID), ({"V": 2 ** 31}, RANGE),
    ({"dtype": 3}, INVALID), ({"logits": None}, INVALID), ({"beam_scores": None}, INVALID),
    ({"token_ids": None}, INVALID), ({"parents": None}, INVALID), ({"scores": None}, INVALID),
    ({"rows": 7}, INVALID), ({"rows": 0}, INVALID), ({"rows": 0, "target": P}, INVALID),
    ({"stride": -1}, INVALID), ({"ws": None}, WORKSPACE), ({"ws_bytes": 8}, WORKSPACE),
    ({"ws": P + 4}, WORKSPACE), ({"G": 2 ** 24, "rows": 2 ** 26}, RANGE)])
def test_select_refusals(change, status):
    assert select(**change) == status


def test_empty_calls():
    assert select(G=0, logits=None) == 0
    assert nat.lib().mvsd_beam_reorder(None, 0, None, None, None, None, 3, 4, None) == 0
    assert nat.lib().mvsd_beam_reorder(None, 3, None, None, None, None, 0, 4, None) == 0


def step_args(**change):
    a = nat.BeamStepArgs()
    for name, kind in nat.BeamStepArgs._fields_:
        if kind is ctypes.c_void_p:
            setattr(a, name, P)
    a.target_rows = None
    a.stride, a.num_rows, a.num_groups, a.beam_width, a.vocab_size = 100, 8, 2, 4, 100
    a.max_length, a.num_stop_ids, a.length_penalty, a.workspace_bytes = 16, 1, 1.0, 1 << 20
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,status", [
    ({"max_length": 0}, INVALID), ({"max_length": 2 ** 31}, RANGE), ({"num_stop_ids": -1}, INVALID),
    ({"num_stop_ids": 64}, RANGE), ({"num_stop_ids": 2 ** 62}, RANGE), ({"dtype": 4}, INVALID),
    ({"beam_width": 65}, RANGE), ({"num_rows": 7}, INVALID), ({"workspace": None}, WORKSPACE)]
    + [({f: None}, INVALID) for f in (
        "scores", "lengths", "done", "finished_scores", "finished_beams", "finished_token_ids",
        "finished_lengths", "out_scores", "out_lengths", "out_done", "out_finished_scores",
        "out_finished_beams", "out_finished_token_ids", "out_finished_lengths", "token_history",
        "parent_history", "token_ids", "parents", "stop_token_ids", "logits")])
def test_step_refusals(change, status):
    assert nat.lib().mvsd_beam_step(ctypes.byref(step_args(**change)), None) == status
    assert nat.lib().mvsd_beam_step(None, None) == INVALID


def finish_args(**change):
    a = nat.BeamFinishArgs()
    for name, kind in nat.BeamFinishArgs._fields_:
        if kind is ctypes.c_void_p:
            setattr(a, name, P)
    a.num_groups, a.beam_width, a.max_length, a.num_return = 2, 4, 16, 4
    a.workspace_bytes = 1 << 20
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,status", [
    ({"num_groups": -1}, INVALID), ({"beam_width": 0}, INVALID), ({"num_return": 0}, INVALID),
    ({"num_return": 5}, INVALID), ({"max_length": 0}, INVALID), ({"max_length": 2 ** 31}, RANGE),
    ({"beam_width": 65}, RANGE), ({"num_groups": 2 ** 40}, RANGE), ({"num_groups": 0}, 0)]
    + [({"max_length": 9000, "workspace": None}, WORKSPACE),
       ({"max_length": 9000, "workspace_bytes": 9}, WORKSPACE),
       ({"num_groups": 2 ** 23}, RANGE), ({"num_groups": 2 ** 12, "max_length": 2 ** 22}, RANGE)]
    + [({f: None}, INVALID) for f, kind in nat.BeamFinishArgs._fields_
       if kind is ctypes.c_void_p and f != "workspace"])
def test_finish_refusals(change, status):
    assert nat.lib().mvsd_beam_finish(ctypes.byref(finish_args(**change)), None) == status
    assert nat.lib().mvsd_beam_finish(None, None) == INVALID


def reorder(states, G=2, W=4, parents=P, slots=None):
    flat = [v for s in states for v in s]
    return nat.lib().mvsd_beam_reorder((ctypes.c_int64 * len(flat))(*flat), len(states), parents,
                                       None, None, slots, G, W, None)


# src, dst, src_stride, dst_stride, num_rows, outer, length, inner: rows of 1024 bytes
GOOD = (P, P, 1024, 1024, 8, 2, 16, 32)


def change(**kw):
    names = ("src", "dst", "src_stride", "dst_stride", "num_rows", "outer", "length", "inner")
    return tuple(kw.get(n, v) for n, v in zip(names, GOOD))


@pytest.mark.parametrize("states,status", [
    ([change(src=0, dst=0)], INVALID), ([change(dst=0)], INVALID), ([change(num_rows=7)], INVALID),
    ([change(num_rows=0)], INVALID), ([change(outer=-1)], INVALID), ([change(length=-1)], INVALID),
    ([change(inner=-1)], INVALID), ([change(src_stride=1023, dst_stride=1023)], INVALID),
    ([change(dst_stride=2048)], INVALID),  # in place with two strides
    ([change(num_rows=2 ** 31)], RANGE), ([change(length=2 ** 31)], RANGE),
    ([change(outer=2 ** 40)], RANGE), ([change(inner=2 ** 62)], RANGE),
    ([change(outer=2 ** 20, inner=2 ** 20)], RANGE),
    ([change(src_stride=2 ** 40, dst_stride=2 ** 40)], RANGE),
    ([GOOD, change(dst=P + 2 ** 16)], INVALID),        # one in place, one not
    ([GOOD, GOOD], INVALID),                            # the same rows twice
    ([GOOD, change(src=P + 512, dst=P + 512)], INVALID),
    ([change(dst=P + 4096)], INVALID),                  # out overlaps the states
    ([change(dst=P + 2 ** 16), change(src=P + 2 ** 17, dst=P + 2 ** 16 + 64)], INVALID),
    ([change(dst=P + 2 ** 16), change(src=P + 2 ** 16 + 1024, dst=P + 2 ** 18)], INVALID),
    ([GOOD] * 513, RANGE)])
def test_reorder_refusals(states, status):
    assert reorder(states) == status


@pytest.mark.parametrize("kw,status", [({"W": 0}, INVALID), ({"W": 65}, RANGE), ({"G": -1}, INVALID),
                                       ({"G": 2 ** 40}, RANGE), ({"parents": None}, INVALID)])
def test_reorder_argument_refusals(kw, status):
    assert reorder([GOOD], **kw) == status


def test_python_refuses_cpu_tensors():
    x, s = torch.zeros(4, 10), torch.zeros(1, 4)
    with pytest.raises(NotImplementedError):
        beam_search_select(x, s, 8)
    state = BeamState.new(1, 4, 8, "cpu")
    with pytest.raises(NotImplementedError):
        beam_search_step(x, state)
    with pytest.raises(NotImplementedError):
        beam_search_finish(state)
    with pytest.raises(NotImplementedError):
        reorder_beams(torch.zeros(4, 8), torch.zeros(1, 4, dtype=torch.int32))


def test_search_arguments():
    for bad in (dict(beam_width=0), dict(beam_width=65), dict(max_length=0),
                dict(beam_width=64, stop_token_ids=[1, 2, 3, 4])):
        args = dict(num_groups=1, beam_width=4, max_length=8, device="cpu", **{})
        args.update(bad)
        with pytest.raises(ValueError):
            BeamSearch(**args)
    search = BeamSearch(2, 4, 8, "cpu", stop_token_ids=[3])
    assert search.state.scores.tolist()[1][0] == 0.0
    assert torch.isneginf(search.state.scores[:, 1:]).all()
    with pytest.raises(RuntimeError):
        search.reorder(torch.zeros(8, 8))


def test_tensor_table_takes_what_fits_and_names_the_first_that_does_not():
    x, y = torch.zeros(3, 4), torch.zeros(5, dtype=torch.int32)
    buf = (ctypes.c_int64 * 4)()
    cpu = x.device

    def table(tensors, dtypes=(torch.float32, torch.int32), shapes=((3, 4), (5,)), at=1,
              device=cpu):
        return _hostops.tensor_table(buf, at, tensors, dtypes, shapes, device)

    assert table((x, y)) == -1
    assert list(buf) == [0, x.data_ptr(), y.data_ptr(), 0]
    assert table((x, y), dtypes=(torch.float32, torch.int64)) == 1
    assert table((x, y), shapes=((4, 3), (5,))) == 0
    assert table((x, y), shapes=((3, 4), (6,))) == 1
    assert table((x, y), device=torch.device("cuda", 0)) == 0
    assert table((x.t(), y), shapes=((4, 3), (5,))) == 0
    assert table((x, None)) == 1 and table((3, y)) == 0
    for bad in (dict(at=3), dict(at=-1), dict(dtypes=(torch.float32,)), dict(shapes=())):
        with pytest.raises(ValueError):
            table((x, y), **bad)
    with pytest.raises(TypeError):
        table([x, y])


def test_state_table_lists_rows_pieces_and_entries():
    x = torch.zeros(6, 3, 10, 4, dtype=torch.float16)
    buf = (ctypes.c_int64 * 24)()
    cpu = x.device

    def table(states, outs=None, dim=2, device=cpu, least=6):
        return _hostops.state_table(buf, states, states if outs is None else outs, dim, device, least)

    assert table((x, x[:, :0], x[:, 1:2])) == 2  # the empty one has no entry
    p = x.data_ptr()
    assert list(buf)[:16] == [p, p, 240, 240, 6, 3, 10, 8, p + 80, p + 80, 240, 240, 6, 1, 10, 8]
    assert table((x,), dim=3) == 1 and list(buf)[4:8] == [6, 30, 4, 2]
    y = torch.zeros(12, 3, 10, 4, dtype=torch.float16)[::2]
    assert table((x,), (y,)) == 1 and list(buf)[:4] == [p, y.data_ptr(), 240, 480]
    for bad in (dict(states=(x,), least=7), dict(states=(x,), dim=4), dict(states=(x,), dim=0),
                dict(states=(x.transpose(1, 2),)), dict(states=(x[..., ::2],)),
                dict(states=(x,), outs=(x.float(),)), dict(states=(x,), outs=(x[:5],)),
                dict(states=(x,), outs=(x, x)), dict(states=(None,)), dict(states=(x, 3)),
                dict(states=(x,), device=torch.device("cuda", 0)),
                dict(states=(x.new_zeros(1, 3, 10, 4).expand(6, 3, 10, 4),)),
                dict(states=(x,) * 4)):
        assert table(**bad) == -1, bad


@pytest.mark.parametrize("alpha", [float("nan"), float("inf"), -float("inf")])
def test_length_penalties_are_finite(alpha):
    assert nat.lib().mvsd_beam_step(ctypes.byref(step_args(length_penalty=alpha, workspace=None)),
                                    None) == INVALID
    assert nat.lib().mvsd_beam_finish(ctypes.byref(finish_args(length_penalty=alpha,
                                                               max_length=9000, workspace=None)),
                                      None) == INVALID


def test_finish_workspace_alignment():
    assert nat.lib().mvsd_beam_finish(ctypes.byref(finish_args(max_length=9000, workspace=P + 2)),
                                      None) == WORKSPACE


def test_the_example_ends_when_no_group_gets_done():
    """The module's example, run on a search whose groups rest at max_length with their flags unset."""
    import textwrap

    from mvsd.sample import beam_search

    lines = beam_search.__doc__.splitlines()
    first = next(k for k, line in enumerate(lines) if line.startswith("    search ="))
    last = next(k for k, line in enumerate(lines) if line.startswith("    answers ="))
    calls = {"step": 0, "finish": 0}

    class Search:
        def __init__(self, *args, **kw):
            self.state = BeamState.new(2, 3, 5, "cpu")

        def step(self, logits):
            calls["step"] += 1
            assert calls["step"] <= 5, "a step after max_length"
            return beam_search.BeamStep(torch.zeros(2, 3), torch.zeros(2, 3), self.state)

        def reorder(self, states, **where):
            return states

        def finish(self, n):
            calls["finish"] += 1

    names = dict(BeamSearch=Search, G=2, W=3, max_length=5, device="cpu", eos=0, n=1, caches=[],
                 prefill=lambda *a: None, decode=lambda *a: None, all_done=False)
    exec(textwrap.dedent("\n".join(lines[first:last + 1])), names)
    assert calls == {"step": 5, "finish": 1}


def test_the_package_is_imported_without_the_host_extension():
    """As libmvsd.so, it is looked for when a call needs it."""
    import sys

    code = ("import sys\n"
            "class Absent:\n"
            "    def find_spec(self, name, path=None, target=None):\n"
            "        if name == 'mvsd._hostops':\n"
            "            raise ImportError(name)\n"
            "sys.meta_path.insert(0, Absent())\n"
            "import mvsd.sample\n"
            "assert 'mvsd._hostops' not in sys.modules\n"
            "import torch\n"
            "state = mvsd.sample.BeamState.new(1, 2, 4, 'cpu')\n"
            "print('imported')\n")
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True,
                          cwd=HEADER.parents[1] / "vllm-from-scratch_amd")
    assert done.returncode == 0 and done.stdout == "imported\n", done.stderr[-500:]
