"""The losses' oracle (oracle/losses.py): its gradients against differences of its values, and values
against their definitions written out."""

import math

import numpy as np
import pytest

from oracle import losses as oracle

EPS = 1e-5  # central differences: error of order EPS^2 against rounding of order 1e-16 / EPS


def differences(f, x):
    out = np.empty(len(x))
    for j in range(len(x)):
        a, b = x.copy(), x.copy()
        a[j] += EPS
        b[j] -= EPS
        out[j] = (f(a) - f(b)) / (2 * EPS)
    return out


@pytest.mark.parametrize("T", [1.0, 0.7])
@pytest.mark.parametrize("g,gH", [(1.0, 0.0), (0.3, -0.8), (0.0, 2.0)])
def test_token_gradient(T, g, gH):
    x = np.random.default_rng(0).normal(size=9) * 2

    def f(x):
        lp, H, _ = oracle.token_row(x, 4, T)
        return g * lp + gH * H

    grad, _ = oracle.token_gradient(oracle.log_softmax(x, T), 4, g, gH, T)
    assert np.allclose(grad, differences(f, x), atol=1e-8)


@pytest.mark.parametrize("ids", [[2], [5, 0, 7], [3, 3, 1, -1], [0, 1, 2, 3, 4, 5, 6, 7]])
@pytest.mark.parametrize("how,tail", [("forward", True), ("forward", False), ("reverse", True),
                                      ("js", True)])
def test_distillation_gradient(ids, how, tail):
    r = np.random.default_rng(len(ids))
    x = r.normal(size=8) * 2
    teacher = oracle.log_softmax(r.normal(size=8))[np.maximum(ids, 0)]

    def f(x):
        return oracle.distill_row(x, ids, teacher, how, tail, 0.8)[0]

    _, grad, _, _ = oracle.distill_row(x, ids, teacher, how, tail, 0.8)
    assert np.allclose(grad, differences(f, x), atol=1e-7)


def test_distillation_from_itself_is_zero():
    x = np.random.default_rng(3).normal(size=11)
    logp = oracle.log_softmax(x)
    for how in ("forward", "reverse", "js"):
        loss, grad, _, _ = oracle.distill_row(x, [4, 9, 1], logp[[4, 9, 1]], how)
        assert abs(loss) < 1e-12 and np.abs(grad).max() < 1e-12


def test_distillation_over_the_whole_vocabulary():
    r = np.random.default_rng(4)
    x, t = r.normal(size=5), oracle.log_softmax(r.normal(size=5))
    q, logp = np.exp(t), oracle.log_softmax(x)
    assert math.isclose(oracle.distill_row(x, range(5), t, "forward")[0], (q * (t - logp)).sum())
    p = np.exp(logp)
    assert math.isclose(oracle.distill_row(x, range(5), t, "reverse")[0], (p * (logp - t)).sum())


@pytest.mark.parametrize("old,A,ref,ent", [(-1.5, 0.7, None, 0.0), (-1.9, -0.7, -1.2, 0.0),
                                           (-1.0, 1.3, -2.0, 0.1), (-2.5, 1.0, -1.0, 0.0),
                                           (-1.0, -1.0, None, 0.0)])
def test_policy_derivative(old, A, ref, ent):
    lp = -1.6
    args = (old, A, ref, 0.2, 0.3, 0.5, ent)
    up = oracle.policy_value(lp + EPS, 1.1, *args)[0]
    down = oracle.policy_value(lp - EPS, 1.1, *args)[0]
    assert abs(oracle.policy_value(lp, 1.1, *args)[1] - (up - down) / (2 * EPS)) < 1e-8


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "squared"])
@pytest.mark.parametrize("m", [-30.0, -1.0, 0.5, 7.0, 40.0])
def test_pair_derivative(kind, m):
    args = (kind, 0.2, 0.1, 0.1 if kind == "sigmoid" else 0.0)
    up, down = oracle.pair_value(m + EPS, *args)[0], oracle.pair_value(m - EPS, *args)[0]
    assert abs(oracle.pair_value(m, *args)[1] - (up - down) / (2 * EPS)) < 1e-7


def test_rows_without_a_distribution():
    for bad in ([NAN, 1.0], [math.inf, 1.0], [-math.inf, -math.inf]):
        assert np.isnan(oracle.log_softmax(bad)).all()
    assert oracle.distill_row([0.0, 1.0], [-1, -1], [0.0, 0.0]) is None


NAN = math.nan
