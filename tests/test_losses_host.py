"""Training losses without a GPU: the C ABI's refusals and struct layout, the Python layer's refusals."""

import ctypes
import subprocess
import threading
from pathlib import Path

import pytest
import torch

from mvsd import _native as nat
from mvsd.sample import distillation_loss, losses, policy_loss, preference_loss, token_logprobs

HEADER = Path(__file__).resolve().parents[1] / "include" / "mvsd.h"
INVALID, WORKSPACE, RANGE = -1, -3, -5
P = 1 << 20  # an address that no refused call touches
LOGPROBS, DISTILL, POLICY, PREFERENCE = range(4)


def test_struct_layout(tmp_path):
    fields = [f for f, _ in nat.LossArgs._fields_]
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){",
             'printf("%zu\\n", sizeof(mvsd_loss_args));']
    lines += [f'printf("%zu\\n", offsetof(mvsd_loss_args, {f}));' for f in fields] + ["return 0;}"]
    (tmp_path / "probe.c").write_text("\n".join(lines))
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-o", str(exe), str(tmp_path / "probe.c")], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    assert got == [ctypes.sizeof(nat.LossArgs)] + [getattr(nat.LossArgs, f).offset for f in fields]


def args(base=POLICY, **change):
    a = nat.LossArgs()
    for name, t in nat.LossArgs._fields_:
        if t is ctypes.c_void_p:
            setattr(a, name, P)
    a.kind, a.ids_dtype, a.reduction, a.tail = base, nat.I32, 1, 1
    a.stride, a.inner_rows, a.num_rows, a.vocab_size, a.temperature = 100, 8, 8, 100, 1.0
    a.num_teacher, a.num_pairs, a.beta, a.clip_low, a.clip_high = 4, 2, 0.1, 0.2, 0.2
    a.workspace_bytes = 1 << 20
    for k, v in change.items():
        setattr(a, k, v)
    return a


BOTH = [
    (POLICY, {"kind": 4}, INVALID), (POLICY, {"kind": -1}, INVALID),
    (POLICY, {"dtype": 3}, INVALID), (POLICY, {"ids_dtype": 0}, INVALID),
    (POLICY, {"logits": None}, INVALID), (POLICY, {"token_ids": None}, INVALID),
    (POLICY, {"num_rows": -1}, INVALID), (POLICY, {"vocab_size": 0}, INVALID),
    (POLICY, {"vocab_size": 2 ** 31}, RANGE), (POLICY, {"num_rows": 2 ** 24}, RANGE),
    (POLICY, {"num_rows": 2 ** 62}, RANGE), (POLICY, {"vocab_size": 2 ** 30, "num_rows": 2048}, RANGE),
    (POLICY, {"inner_rows": 0}, INVALID), (POLICY, {"stride": -1}, INVALID),
    (POLICY, {"outer_stride": -1}, INVALID), (POLICY, {"temperature": 0.0}, INVALID),
    (POLICY, {"temperature": float("nan")}, INVALID), (POLICY, {"temperature": 1e9}, INVALID),
    (POLICY, {"reduction": 3}, INVALID), (POLICY, {"advantages": None}, INVALID),
    (POLICY, {"saved": P + 4}, WORKSPACE),
    (DISTILL, {"num_teacher": 0}, INVALID), (DISTILL, {"num_teacher": 513}, RANGE),
    (DISTILL, {"teacher_logprobs": None}, INVALID), (DISTILL, {"divergence": 3}, INVALID),
    (DISTILL, {"divergence": 1, "tail": 0}, INVALID), (DISTILL, {"divergence": 2, "tail": 0}, INVALID),
    (PREFERENCE, {"loss_type": 3}, INVALID), (PREFERENCE, {"num_pairs": -1}, INVALID),
    (PREFERENCE, {"num_pairs": 2 ** 40}, RANGE), (PREFERENCE, {"num_pairs": 2 ** 23 + 1}, RANGE),
    (PREFERENCE, {"cu_num_tokens": None, "num_pairs": 3}, INVALID),
    (PREFERENCE, {"loss_type": 2, "beta": 0.0}, INVALID),
]


@pytest.mark.parametrize("kind,change,status", BOTH)
def test_refusals_of_both_calls(kind, change, status):
    a = args(kind, **change)
    assert nat.lib().mvsd_row_loss(ctypes.byref(a), None) == status
    assert nat.lib().mvsd_loss_gradient(ctypes.byref(a), P, 0, None, 0, None) == status


@pytest.mark.parametrize("kind,change,status", [
    (POLICY, {"loss": None}, INVALID), (DISTILL, {"loss": None}, INVALID),
    (DISTILL, {"loss": None, "reduction": 2}, INVALID), (PREFERENCE, {"loss": None}, INVALID),
    (LOGPROBS, {"logprobs": None}, INVALID), (POLICY, {"logprobs": None}, INVALID),
    (PREFERENCE, {"logprobs": None}, INVALID), (POLICY, {"workspace": None}, WORKSPACE),
    (POLICY, {"workspace_bytes": 8}, WORKSPACE), (POLICY, {"workspace": P + 8}, WORKSPACE)])
def test_refusals_of_the_values(kind, change, status):
    assert nat.lib().mvsd_row_loss(ctypes.byref(args(kind, **change)), None) == status


@pytest.mark.parametrize("kind,change,up,status", [
    (POLICY, {"grad": None}, (P, 0, None, 0), INVALID), (POLICY, {}, (None, 0, None, 0), INVALID),
    (POLICY, {}, (P, -1, None, 0), INVALID), (LOGPROBS, {}, (P, 0, P, -1), INVALID),
    (POLICY, {"saved": None}, (P, 0, None, 0), WORKSPACE)])
def test_refusals_of_the_gradient(kind, change, up, status):
    assert nat.lib().mvsd_loss_gradient(ctypes.byref(args(kind, **change)), *up, None) == status


@pytest.mark.parametrize("kind,change", [
    (POLICY, {}), (POLICY, {"num_rows": 4096, "reduction": 2}), (DISTILL, {}), (PREFERENCE, {}),
    (LOGPROBS, {"num_rows": 4096, "vocab_size": 50257})])
def test_a_gradient_that_no_call_wrote(kind, change):
    """Only values of one pass write the gradient of an upstream of 1."""
    a = args(kind, unit_gradient=1, **change)
    assert nat.lib().mvsd_loss_one_pass(ctypes.byref(a)) == 0
    assert nat.lib().mvsd_loss_gradient(ctypes.byref(a), P, 0, None, 0, None) == INVALID


def test_null_arguments():
    lib = nat.lib()
    assert lib.mvsd_row_loss(None, None) == INVALID
    assert lib.mvsd_loss_gradient(None, P, 0, None, 0, None) == INVALID
    assert lib.mvsd_loss_workspace_bytes(None) == INVALID
    assert lib.mvsd_loss_saved_bytes(None) == INVALID


def test_sizes():
    lib = nat.lib()
    small = lib.mvsd_loss_workspace_bytes(ctypes.byref(args(num_rows=1)))
    large = lib.mvsd_loss_workspace_bytes(ctypes.byref(args(num_rows=4096, vocab_size=151936)))
    assert 0 < small < large
    # a pair's place, also where there are more pairs than rows
    few = lib.mvsd_loss_workspace_bytes(ctypes.byref(args(PREFERENCE, num_rows=0, num_pairs=5000)))
    assert few >= 20000
    assert lib.mvsd_loss_saved_bytes(ctypes.byref(args(num_rows=8))) == 8 * 32
    assert lib.mvsd_loss_saved_bytes(ctypes.byref(args(DISTILL, num_rows=8))) == 8 * (32 + 4 * 8)


def test_an_empty_gradient_is_no_work():
    a = args(num_rows=0, logits=None, token_ids=None, grad=None, saved=None)
    assert nat.lib().mvsd_loss_gradient(ctypes.byref(a), P, 0, None, 0, None) == 0


X, IDS, ROWS = torch.zeros(4, 10), torch.zeros(4, dtype=torch.int32), torch.zeros(4)


@pytest.mark.parametrize("call", [
    lambda: token_logprobs(X, IDS),
    lambda: distillation_loss(X, torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)),
    lambda: policy_loss(X, IDS, ROWS, ROWS),
    lambda: preference_loss(X, IDS, cu_num_tokens=torch.tensor([2, 4], dtype=torch.int32))])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(NotImplementedError):
        call()


@pytest.mark.parametrize("call", [
    lambda: distillation_loss(X, IDS[:, None], ROWS[:, None], reduction="total"),
    lambda: policy_loss(X, IDS, ROWS, ROWS, reduction=None),
    lambda: preference_loss(X, IDS, reduction=["mean"])])
def test_unknown_reductions_are_refused(call):
    with pytest.raises(ValueError, match="reduction"):
        call()


# --------------------------------------------------------------------------- backward passes


class Entry:
    """Stands in for the gradient's C entry: two calls at once, each of which writes its upstream's index
    where its own arguments point to when both are inside."""

    def __init__(self):
        self.both = threading.Barrier(2, timeout=20)

    def mvsd_loss_gradient(self, ref, up, *more):
        a = ref._obj
        self.both.wait()
        value = ctypes.c_float.from_address(up).value
        ctypes.c_float.from_address(a.grad).value = value
        ctypes.c_float.from_address(a.grad + 4).value = float(a.unit_gradient)
        self.both.wait()
        return 0


def test_two_backward_passes_at_once(monkeypatch):
    """Over one kept graph, as threads make them where the engine has none of its own: each writes its own
    gradient, and only one of them has the one that is there already."""
    entry = Entry()
    monkeypatch.setattr(nat, "lib", lambda: entry)
    monkeypatch.setattr(nat, "stream_of", lambda device: 0)
    call = losses._Call.__new__(losses._Call)
    x, ids, saved = torch.zeros(2, 3), torch.zeros(2, dtype=torch.int32), torch.zeros(8)
    call.args, call.kind, call.layout, call.fresh = args(), POLICY, (x.data_ptr(), x.stride()), [True]
    unit = torch.zeros(2, 3)
    for units in ([0.0, 1.0], [0.0, 0.0]):
        got = {}

        def back(n):
            got[n] = call.gradient(x, ids, saved, unit, torch.tensor(float(n)), None)

        threads = [threading.Thread(target=back, args=(n,)) for n in (1, 2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert [float(got[n][0, 0]) for n in (1, 2)] == [1.0, 2.0]
        assert sorted(float(got[n][0, 1]) for n in (1, 2)) == units


def test_forward_mode_is_refused():
    """A tangent of the logits is not dropped, whether or not they want a gradient as well."""
    import torch.autograd.forward_ad as forward_ad

    class Stub:
        def __init__(self, logits):
            self.logits, self.outputs = logits, (logits.detach(),)

        def run(self, train):
            pass

    assert losses._finish(Stub(X))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(X.clone(), torch.ones_like(X))
        with pytest.raises(NotImplementedError):
            losses._finish(Stub(dual))
        with torch.no_grad(), pytest.raises(NotImplementedError):
            losses._finish(Stub(dual))
        assert losses._finish(Stub(dual.detach()))


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("kind,name", [
    (POLICY, "clip_low"), (POLICY, "clip_high"), (POLICY, "kl_coef"), (POLICY, "entropy_coef"),
    (PREFERENCE, "beta"), (PREFERENCE, "margin"), (PREFERENCE, "label_smoothing")])
@pytest.mark.parametrize("loss_type", [0, 1, 2])
def test_numbers_that_are_not_finite(kind, name, value, loss_type):
    """Refused before anything is launched: the workspace is one that no call takes."""
    a = args(kind, loss_type=loss_type, workspace=None, saved=None)
    assert nat.lib().mvsd_row_loss(ctypes.byref(a), None) == WORKSPACE
    assert nat.lib().mvsd_loss_gradient(ctypes.byref(a), P, 0, None, 0, None) == WORKSPACE
    setattr(a, name, value)
    assert nat.lib().mvsd_row_loss(ctypes.byref(a), None) == INVALID
    assert nat.lib().mvsd_loss_gradient(ctypes.byref(a), P, 0, None, 0, None) == INVALID
