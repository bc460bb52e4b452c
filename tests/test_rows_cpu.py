"""Host checks of the row operators: refusals before any device call, and the oracle itself."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import rows_oracle as oracle
import torch

import povs
from povs import _native


@pytest.mark.parametrize("call", [
    lambda: povs.sample(torch.zeros(2, 3), torch.zeros(2)),
    lambda: povs.sample([[1.0]], torch.zeros(1)),
    lambda: povs.route(torch.zeros(2, 3), 1),
    lambda: povs.plan_rows(torch.zeros(2, 3, dtype=torch.int32), 3),
    lambda: povs.dispatch_rows(torch.zeros(2, 3), povs.RowPlan(*[torch.zeros(2, 1, dtype=torch.int32)] * 3)),
    lambda: povs.combine_rows(np.zeros((2, 3)), povs.RowPlan(*[torch.zeros(2, 1, dtype=torch.int32)] * 3)),
])
def test_host_tensors_are_refused(call):
    with pytest.raises(TypeError):
        call()




def _sample(**kw):
    a = dict(logits=64, dtype=0, rows=2, width=8, stride=8, u=64, ub=4, ts=None, t=1.0, ks=None, k=0, ps=None, p=1.0,
             ms=None, m=0.0, ids=64, device=0, stream=None)
    a.update(kw)
    return _native.load().povs_sample_v1(*a.values())


@pytest.mark.parametrize("kw,code,says", [
    (dict(logits=None), -1, b"NULL"), (dict(u=None), -1, b"NULL"), (dict(ids=None), -1, b"NULL"),
    (dict(dtype=3), -1, b"dtype"), (dict(rows=-1), -1, b"rows"), (dict(width=0), -1, b"width"),
    (dict(width=2**31), -2, b"2^31"), (dict(ub=2), -1, b"uniform_bytes"), (dict(t=-1.0), -1, b"temperature"),
    (dict(t=float("nan")), -1, b"temperature"), (dict(t=float("inf")), -1, b"temperature"), (dict(k=-1), -1, b"top_k"),
    (dict(p=1.5), -1, b"top_p"), (dict(p=float("nan")), -1, b"top_p"), (dict(m=-0.1), -1, b"min_p"),
    (dict(device=99), -1, b"device"), (dict(device=-1), -1, b"device"),
])
def test_sample_refusals(kw, code, says):
    assert _sample(**kw) == code
    assert says in _native.load().povs_last_error_string()


def _route(**kw):
    a = dict(logits=64, dtype=0, rows=2, n=16, stride=16, bias=None, k=2, scoring=0, groups=1, top_groups=1, gs=0,
             renorm=0, scale=1.0, experts=64, weights=64, device=0, stream=None)
    a.update(kw)
    return _native.load().povs_route_v1(*a.values())


@pytest.mark.parametrize("kw,code,says", [
    (dict(logits=None), -1, b"logits"), (dict(experts=None), -1, b"experts"), (dict(weights=None), -1, b"weights"),
    (dict(dtype=-1), -1, b"dtype"), (dict(rows=-1), -1, b"rows"), (dict(n=0), -1, b"n_experts"),
    (dict(n=1025), -2, b"limit"), (dict(k=0), -1, b"top_k"), (dict(k=17), -1, b"top_k"),
    (dict(n=64, k=33), -2, b"top_k"), (dict(scoring=2), -1, b"scoring"), (dict(gs=5), -1, b"group_score"),
    (dict(groups=3), -1, b"n_groups"), (dict(groups=0), -1, b"n_groups"), (dict(n=64, groups=64, top_groups=4), -2, b"groups"),
    (dict(groups=4, top_groups=5), -1, b"top_groups"), (dict(groups=4, top_groups=0), -1, b"top_groups"),
    (dict(groups=8, top_groups=1, k=3), -1, b"top_k"), (dict(scale=float("inf")), -1, b"scale"),
    (dict(rows=2**30), -2, b"rows"), (dict(device=64), -1, b"device"),
])
def test_route_refusals(kw, code, says):
    assert _route(**kw) == code
    assert says in _native.load().povs_last_error_string()


def test_route_backward_refusals():
    lib = _native.load()
    good = [64, 0, 2, 16, 16, 2, 0, 0, 1.0, 64, 64, 64, 0, None]
    for at, value in ((0, None), (1, 9), (2, -1), (3, 0), (5, 0), (6, 7), (9, None), (10, None), (11, None), (12, -3)):
        args = list(good)
        args[at] = value
        assert lib.povs_route_backward_v1(*args) == -1, at


def test_plan_refusals_and_workspace():
    lib = _native.load()
    assert lib.povs_plan_rows_workspace_v1(-1, 4) == -1
    assert lib.povs_plan_rows_workspace_v1(10, 0) == -1
    assert lib.povs_plan_rows_workspace_v1(10, 4097) == -2
    assert lib.povs_plan_rows_workspace_v1(2**31, 4) == -2
    assert lib.povs_plan_rows_workspace_v1(0, 4) == 0 and lib.povs_plan_rows_workspace_v1(100, 4) == 0
    need = lib.povs_plan_rows_workspace_v1(1 << 20, 256)
    assert need > 0
    good = [64, 4, 1 << 20, 256, 64, 64, 64, 64, need, 0, None]
    for at, value in ((0, None), (1, 2), (2, -1), (3, 0), (4, None), (5, None), (6, None), (7, None), (8, need - 1), (9, -1)):
        args = list(good)
        args[at] = value
        assert lib.povs_plan_rows_v1(*args) == -1, at


def test_dispatch_and_combine_refusals():
    lib = _native.load()
    good = [64, 4, 16, 16, 64, 2, 64, 64, 8, 0, None]
    for at, value, code in ((0, None, -1), (1, -1, -1), (2, -1, -1), (3, -1, -1), (4, None, -1), (5, 0, -1), (6, None, -1),
                            (7, None, -1), (8, -1, -1), (8, 2**31, -2), (1, 2**31, -2), (9, 64, -1)):
        args = list(good)
        args[at] = value
        assert lib.povs_dispatch_rows_v1(*args) == code, at
    good = [64, 0, 8, 16, 16, 64, 4, 2, None, 64, 0, None]
    for at, value, code in ((0, None, -1), (1, 4, -1), (2, -1, -1), (3, -1, -1), (4, -1, -1), (5, None, -1), (6, -1, -1),
                            (7, 0, -1), (9, None, -1), (10, -1, -1), (2, 2**31, -2)):
        args = list(good)
        args[at] = value
        assert lib.povs_combine_rows_v1(*args) == code, at
    good = [64, 64, 1, 8, 16, 16, 64, 4, 2, None, 64, 64, 64, 0, None]
    for at, value, code in ((0, None, -1), (1, None, -1), (2, 7, -1), (3, -1, -1), (6, None, -1), (8, 0, -1), (10, None, -1),
                            (13, 99, -1), (7, 2**31, -2)):
        args = list(good)
        args[at] = value
        assert lib.povs_combine_backward_v1(*args) == code, at


def test_nothing_to_do_needs_no_device():
    lib = _native.load()
    assert lib.povs_sample_v1(None, 0, 0, 8, 8, None, 4, None, 1.0, None, 0, None, 1.0, None, 0.0, None, 0, None) == 0
    assert lib.povs_dispatch_rows_v1(None, 0, 16, 16, None, 2, None, None, 0, 0, None) == 0
    assert lib.povs_combine_rows_v1(None, 0, 0, 16, 16, None, 0, 2, None, None, 0, None) == 0


def test_the_oracle_draws_what_its_rules_say():
    x = np.log(np.array([1.0, 4.0, 2.0, 0.0, 3.0], dtype=np.float64), where=np.array([1, 1, 1, 0, 1], bool),
               out=np.full(5, -np.inf))
    assert [oracle.sample_row(x, u) for u in (0.0, 0.099, 0.101, 0.499, 0.501, 0.699, 0.701, 0.999)] == [0, 0, 1, 1, 2, 2, 4, 4]
    assert {oracle.sample_row(x, u, top_k=2) for u in np.linspace(0, 0.999, 50)} == {1, 4}
    assert {oracle.sample_row(x, u, top_p=0.4) for u in np.linspace(0, 0.999, 50)} == {1}
    assert {oracle.sample_row(x, u, top_p=0.71) for u in np.linspace(0, 0.999, 50)} == {1, 2, 4}
    assert {oracle.sample_row(x, u, min_p=0.5) for u in np.linspace(0, 0.999, 50)} == {1, 2, 4}
    assert oracle.sample_row(x, 0.9, temperature=0.0) == 1
    assert oracle.sample_row(np.full(4, -np.inf), 0.5) == -1


def test_the_oracle_routes_what_its_rules_say():
    x = np.array([0.0, 1.0, 1.0, -np.inf, 3.0, 2.0])
    e, w = oracle.route_row(x, 4)
    assert e.tolist() == [4, 5, 1, 2] and w[0] > w[1] > w[2] == w[3]
    e, w = oracle.route_row(x, 6, renormalize=True)
    assert e.tolist() == [4, 5, 1, 2, 0, -1] and w[5] == 0 and abs(w.sum() - 1) < 1e-15
    e, _ = oracle.route_row(x, 2, n_groups=3, top_groups=1, group_score="max")
    assert e.tolist() == [4, 5]
    e, _ = oracle.route_row(x, 2, n_groups=3, top_groups=2, bias=np.array([5.0, 5, 0, 0, 0, 0]))
    assert e.tolist() == [1, 0]
    slots, sources, offsets = oracle.plan(np.array([[1, 0], [-1, 1], [0, 2]]), 3)
    assert slots.tolist() == [[2, 0], [-1, 3], [1, 4]] and sources.tolist() == [1, 4, 0, 3, 5, -1] and offsets.tolist() == [0, 2, 4, 5]
