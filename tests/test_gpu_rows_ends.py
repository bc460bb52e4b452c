"""Row operators on the GPU at the ends of what they take: scores that 32 bits lose, masks of finite
value, sums that cancel, random numbers on a border.

Against the definitions in 64 bits (tests/rows_oracle.py); tolerances count roundings as in
tests/test_gpu_rows.py.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import rows_oracle as oracle
import torch

import povs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U32 = 2.0**-24


def _host(t: torch.Tensor) -> np.ndarray:
    t = t.detach().cpu()
    return t.double().numpy() if t.is_floating_point() else t.numpy()


def _randn(*shape, seed: int, sharp: float = 1.0, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * sharp).to(dtype).to(DEV)


def _same_route(x: torch.Tensor, k: int, **kw) -> None:
    host = {**kw, "bias": _host(kw["bias"])} if kw.get("bias") is not None else kw
    experts, _ = oracle.route(_host(x), k, **host)
    np.testing.assert_array_equal(_host(povs.route(x, k, **kw).experts), experts)


# Rows for a warp each, and enough to fill the GPU with lanes.
FEW_AND_MANY = [300, 9600]


@pytest.mark.parametrize("n,groups,top_groups,k,rows", [(64, 8, 4, 6, 300), (96, 32, 9, 4, 300), (512, 16, 3, 10, 300),
                                                        (64, 8, 4, 12, 9600), (256, 8, 4, 8, 9600)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_route_groups_with_nan_scores(dtype, n, groups, top_groups, k, rows):
    """A NaN logit ranks below every number of its group, wherever in the group it stands."""
    x = _randn(rows, n, seed=n, sharp=0.5, dtype=dtype)
    at = torch.randint(0, n, (rows, 2), generator=torch.Generator().manual_seed(1)).to(DEV)
    x.scatter_(1, at, float("nan"))
    _same_route(x, k, scoring="sigmoid", n_groups=groups, top_groups=top_groups)


def test_route_groups_with_nan_biases_and_masks():
    """NaN biases, and groups that masks leave one number or none: those of a number and NaN count no
    more and no less than those of a number and a masked expert."""
    n, groups = 64, 16
    x = _randn(200, n, seed=4, sharp=0.5)
    bias = torch.zeros(n, device=DEV)
    bias[::9] = float("nan")
    _same_route(x, 6, scoring="sigmoid", bias=bias, n_groups=groups, top_groups=5)
    x[:100, :40] = -float("inf")
    x[:50, 3::4] = 0.25
    x[:100, 1::4] = float("nan")
    _same_route(x, 4, scoring="sigmoid", n_groups=groups, top_groups=10)
    _same_route(x, 4, scoring="sigmoid", bias=bias, n_groups=groups, top_groups=12, group_score="max")


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("n,groups,top_groups,k,rows", [(64, 32, 9, 6, 2000), (96, 32, 9, 6, 2000), (256, 32, 9, 6, 9600)])
def test_route_groups_whose_biases_cancel(n, groups, top_groups, k, rows, scoring):
    """Two highest scores of +600 and -600: each is rounded by 2^-15, while groups' sums lie 10^-5 apart."""
    x = _randn(rows, n, seed=n, sharp=0.01)
    bias = torch.full((groups, n // groups), -2000.0, device=DEV)
    bias[:, 0], bias[:, 1] = 600.0, -600.0
    _same_route(x, k, scoring=scoring, bias=bias.reshape(-1), n_groups=groups, top_groups=top_groups)


def _weight_bound(x: np.ndarray, n: int) -> float:
    """Relative error of a weight in 32 bits: the exponential's argument, rounded twice relative to its
    size (a logit, or its difference from the highest), the exponential and the quotients (16 steps), and
    sums over n scores by one lane and over up to 32 chosen ones."""
    finite = x[np.isfinite(x)]
    return (2 * (np.abs(finite).max() + finite.max() - finite.min()) + n + 32 + 16) * U32


@pytest.mark.parametrize("rows", FEW_AND_MANY)
@pytest.mark.parametrize("level", [-27.0, -87.0, -100.0, -300.0])
@pytest.mark.parametrize("dtype,bias", [(torch.float32, False), (torch.float32, True), (torch.bfloat16, False)], ids=str)
def test_route_renormalizes_scores_below_32_bits(dtype, bias, level, rows):
    """Sigmoid scores that 32 bits flush to 0 still have quotients, which sum to the scale.  Where the
    chosen scores' sum is 2^-40 or more, a flushed score is below 2^-86 of it."""
    n, k, scale = 64, 6, 16.0
    x = (_randn(rows, n, seed=5) + level).to(dtype)
    kw = dict(scoring="sigmoid", renormalize=True, scale=scale)
    if bias:
        kw["bias"] = _randn(n, seed=6, sharp=0.1)
    got = povs.route(x, k, **kw)
    experts, weights = oracle.route(_host(x), k, **{**kw, "bias": _host(kw["bias"]) if bias else None})
    np.testing.assert_array_equal(_host(got.experts), experts)
    np.testing.assert_allclose(_host(got.weights), weights, rtol=_weight_bound(_host(x), n), atol=2.0**-86 * scale)
    assert np.abs(_host(got.weights).sum(1) / scale - 1).max() < 1e-4


@pytest.mark.parametrize("rows", FEW_AND_MANY)
def test_route_renormalizes_softmax_scores_below_32_bits(rows):
    """A bias brings experts forward whose softmax scores are e^-100 and less."""
    n, k = 64, 4
    x = _randn(rows, n, seed=7)
    x[:, :8] += 120.0
    bias = _randn(n, seed=8, sharp=0.1)  # so far apart that 32 bits decide
    bias[:8] = -3.0
    got = povs.route(x, k, bias=bias, renormalize=True)
    experts, weights = oracle.route(_host(x), k, bias=_host(bias), renormalize=True)
    assert (experts >= 8).all()
    np.testing.assert_array_equal(_host(got.experts), experts)
    np.testing.assert_allclose(_host(got.weights), weights, rtol=_weight_bound(_host(x), n))


def test_route_scales_of_any_size():
    """Renormalised weights are quotients times the scale, also where score times scale or scale by sum would
    leave 32 bits."""
    x = _randn(200, 32, seed=8) - 20.0
    for scale in (1e-30, 1e36):
        got = povs.route(x, 4, scoring="sigmoid", renormalize=True, scale=scale)
        _, weights = oracle.route(_host(x), 4, scoring="sigmoid", renormalize=True, scale=scale)
        np.testing.assert_allclose(_host(got.weights), weights, rtol=_weight_bound(_host(x), 32))


def _gradient(x, experts, g, scoring, renormalize, scale):
    """(gradient of the logits, the size of the terms whose sum each of its numbers is), in 64 bits.

    With f the scores, w the weights before scaling and j a chosen expert, without a difference of large
    numbers: dx_j = f_j (g_j U + sum_i f_i (g_j - g_i)) for a softmax, U the scores of those not chosen (0
    for quotients); dx_j = f_j (1 - f_j) g_j for a sigmoid, w_j (1 - f_j) sum_i w_i (g_j - g_i) for its
    quotients; dx_i = -s_i sum_j f_j g_j elsewhere in a softmax's row."""
    x, g = x.astype(np.float64), g.astype(np.float64)
    out, size = np.zeros_like(x), np.zeros_like(x)
    for r in range(len(x)):
        e = experts[r][experts[r] >= 0]
        up = g[r][experts[r] >= 0] * scale
        if scoring == "softmax":
            s = np.exp(x[r] - x[r].max())
            s /= s.sum()
            other = np.delete(s, e).sum()
        else:
            s, complement = 1 / (1 + np.exp(-x[r])), 1 / (1 + np.exp(x[r]))
        f = s[e]
        w = f / f.sum() if renormalize else f
        apart = up[:, None] - up[None, :]
        if renormalize:
            d, m = w * (apart @ w), w * (np.abs(apart) @ w)
            if scoring == "sigmoid":
                d, m = d * complement[e], m * complement[e]
        elif scoring == "softmax":
            out[r], size[r] = -s * (f * up).sum(), s * (f * np.abs(up)).sum()
            d, m = f * (up * other + apart @ f), f * (np.abs(up) * other + np.abs(apart) @ f)
        else:
            d = f * complement[e] * up
            m = np.abs(d)
        out[r, e], size[r, e] = d, m
    return out, size


def _gradient_bound(size, want, dtype, x, n):
    """One rounding to the type; in 32 bits each term is a product of up to three scores or weights (each
    with a weight's error) and a difference, summed over up to 32 chosen ones."""
    tiny = {torch.float32: 2.0**-126, torch.bfloat16: 2.0**-126, torch.float16: 2.0**-24}[dtype]
    return torch.finfo(dtype).eps / 2 * np.abs(want) + (3 * _weight_bound(x, n) + 40 * U32) * size + tiny


def _check_gradient(x, k, seed, **kw):
    x = x.detach().requires_grad_()
    experts, weights = povs.route(x, k, **kw)
    g = _randn(*weights.shape, seed=seed)
    (dx,) = torch.autograd.grad(weights, x, g)
    want, size = _gradient(_host(x), _host(experts), _host(g), kw.get("scoring", "softmax"),
                           kw.get("renormalize", False), kw.get("scale", 1.0))
    assert (np.abs(_host(dx) - want) <= _gradient_bound(size, want, x.dtype, _host(x), x.shape[1])).all()
    return dx


@pytest.mark.parametrize("level", [-10.0, -87.0, -100.0, -300.0])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_route_gradient_of_scores_below_32_bits(dtype, level):
    x = (_randn(60, 40, seed=9) + level).to(dtype)
    dx = _check_gradient(x, 5, seed=1, scoring="sigmoid", renormalize=True, scale=2.5)
    assert ((dx != 0).sum(1) >= 4).all()


def test_route_gradient_of_softmax_scores_below_32_bits():
    x = _randn(60, 40, seed=10)
    x[:, :8] += 120.0
    bias = torch.zeros(40, device=DEV)
    bias[:8] = -3.0
    dx = _check_gradient(x, 5, seed=2, bias=bias, renormalize=True)
    assert ((dx != 0).sum(1) >= 4).all()


@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("level", [10.0, 17.0, 30.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=str)
def test_route_gradient_of_sigmoid_scores_near_one(dtype, level, renormalize):
    """The factor 1 - s keeps its relative accuracy where s is rounded to 1."""
    x = (_randn(60, 40, seed=11) + level).to(dtype)
    _check_gradient(x, 5, seed=3, scoring="sigmoid", renormalize=renormalize)


@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("k", [1, 8])
@pytest.mark.parametrize("level", [5.0, 40.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_route_gradient_of_softmax_scores_near_one(dtype, level, k, renormalize):
    """One expert far above the rest: its gradient is a small difference, and is summed without one."""
    x = _randn(60, 48, seed=12)
    x[torch.arange(60), torch.arange(60) % 48] += level
    _check_gradient(x.to(dtype), k, seed=4, renormalize=renormalize)


@pytest.mark.parametrize("score", [0.0, 0.3, 0.235038429])
@pytest.mark.parametrize("width", [131072, 16384])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_sample_constant_rows_at_even_random_numbers(dtype, width, score):
    """Random numbers on the border of two equal ids: one of the two, within the rounding of the sums."""
    n = 1 << 14
    row = torch.full((1, width), score, dtype=dtype, device=DEV)
    u = torch.arange(n, dtype=torch.float64, device=DEV) / n
    ids = torch.cat([povs.sample(row.expand(2048, -1), part) for part in u.split(2048)])
    want = torch.floor(u * width).long()
    assert (ids >= 0).all() and (ids < width).all()
    assert ((ids - want).abs() <= 1).all()


ENDS = [0.0, 2.0**-60, 0.5, 1.0 - 2.0**-24, 1.0 - 2.0**-53, 1.0, 7.5, -1.0, float("nan")]


@pytest.mark.parametrize("kw", [{}, {"temperature": 0.05}, {"top_p": 0.999}, {"top_k": 3000}, {"min_p": 1e-7},
                                {"top_k": 3000, "min_p": 1e-3}], ids=str)
@pytest.mark.parametrize("dtype,mask", [(torch.float32, -1e4), (torch.float32, "lowest"), (torch.float16, "lowest")], ids=str)
@pytest.mark.parametrize("width", [301, 40_009])
def test_sample_masks_of_finite_value_are_never_drawn(width, dtype, mask, kw):
    """Ids masked with a finite score weigh 0 in 64 bits.  Between masked runs at both ends, random numbers at
    and beyond the ends of [0, 1) draw the first or the last id that has a weight."""
    first, last = width // 3, width - width // 4
    x = torch.full((len(ENDS), width), torch.finfo(dtype).min if mask == "lowest" else mask, dtype=dtype)
    x[:, first:last] = torch.linspace(0.0, 1.0, last - first).to(dtype) * 0.01
    x = x.to(DEV)
    for u in (torch.tensor(ENDS, dtype=torch.float64, device=DEV), torch.tensor(ENDS, device=DEV)):
        got = _host(povs.sample(x, u, **kw))
        want = [oracle.sample_row(_host(x[r]), 0.0 if np.isnan(v) else v, **kw) for r, v in enumerate(_host(u))]
        low, high = want[0], want[5]
        assert first <= low <= high < last
        exact = [0, 5, 6, 7, 8]
        assert [got[i] for i in exact] == [want[i] for i in exact]
        assert (got >= low).all() and (got <= high).all()


@pytest.mark.parametrize("kw", [{}, {"top_p": 0.9999}, {"top_k": 30_000}], ids=str)
@pytest.mark.parametrize("width", [500, 40_009])
def test_sample_min_p_at_a_weight(width, kw):
    """A lowest weight 2^-46 above or below that of thousands of equal scores keeps all of them or none."""
    x = torch.where(torch.arange(width) % 3 == 0, 0.0, -2.0).to(torch.float32).expand(40, -1).to(DEV)
    u = ((torch.arange(40, dtype=torch.float64) + 0.5) / 40).to(DEV)
    for min_p in (math.exp(-2.0) * (1 - 2.0**-46), math.exp(-2.0) * (1 + 2.0**-46)):
        got = _host(povs.sample(x, u, min_p=min_p, **kw))
        want = [oracle.sample_row(_host(x[r]), v, min_p=min_p, **kw) for r, v in enumerate(_host(u))]
        np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("kw", [{}, {"top_k": 200}, {"top_k": 2000}, {"top_k": 9000}, {"top_p": 1 - 1e-15}, {"min_p": 1e-200}], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("width", [257, 5000, 40_009])
def test_sample_zero_draws_the_first_weight(width, dtype, kw):
    """At 0 the running sum has to exceed 0: the lowest id with any weight that 64 bits hold."""
    rows = 8
    g = torch.Generator().manual_seed(width)
    x = -torch.rand(rows, width, generator=g) * 0.2
    heavy = torch.randint(width // 2, width, (rows, 1), generator=g)
    x.scatter_(1, heavy, 0.0)
    for temperature, level in ((1.0, 60.0), (0.1, 9.0), (0.01, 6.5)):
        y = (x * 0.1 - level).scatter_(1, heavy, 0.0)
        y[0::2, :3] = -800.0  # weighs nothing at any of the temperatures
        y = y.to(dtype).to(DEV)
        got = _host(povs.sample(y, torch.zeros(rows, device=DEV), temperature=temperature, **kw))
        want = [oracle.sample_row(_host(r), 0.0, temperature=temperature, **kw) for r in y]
        np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("width", [100_003, 1_500_001])
def test_sample_small_weights_of_a_wide_row(width):
    """One id of weight 1 before 1499 of weight e^-25, among scores far below: random numbers in the middle of
    each of the small ones draw it.  Rounded to 2^-51 of the highest, 1499 of them are off by 2^-41 in all, a
    twentieth of one."""
    k = 1500
    g = torch.Generator().manual_seed(1)
    row = -100.0 - 100.0 * torch.rand(width, generator=g)
    at = torch.sort(torch.randperm(width - 1, generator=g)[: k - 1] + 1).values
    row[0], row[at] = 0.0, -25.0
    picks = torch.arange(0, k - 1, 37)
    w = math.exp(-25.0)
    u = (1.0 + (picks.double() + 0.5) * w) / (1.0 + (k - 1) * w)
    for kw in ({"top_k": k}, {"min_p": 1e-12}):
        got = povs.sample(row.to(DEV).expand(len(picks), -1), u.to(DEV), **kw).cpu()
        assert torch.equal(got, at[picks])


def test_forward_mode_differentiation_is_refused():
    """A tangent is refused, as a second-order gradient is, and not dropped."""
    plan = povs.plan_rows(torch.zeros(4, 2, dtype=torch.int32, device=DEV), 3)
    x, y, w = _randn(4, 8, seed=1), _randn(8, 5, seed=2), torch.rand(4, 2, device=DEV)
    with torch.autograd.forward_ad.dual_level():
        def dual(t):
            return torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: povs.route(dual(x), 2), lambda: povs.dispatch_rows(dual(x), plan),
                     lambda: povs.combine_rows(dual(y), plan), lambda: povs.combine_rows(y, plan, dual(w)),
                     lambda: povs.route(dual(x).requires_grad_(), 2)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        assert torch.equal(povs.combine_rows(y, plan, w), povs.combine_rows(y.clone(), plan, w))
        assert povs.route(x, 2).weights.shape == (4, 2)


def test_combine_keeps_rows_for_the_weights_gradient_alone():
    plan = povs.plan_rows(torch.randint(0, 3, (16, 2), device=DEV), 3)
    y = _randn(32, 5, seed=1).requires_grad_()
    w = torch.rand(16, 2, device=DEV)
    for weights, kept in ((None, False), (w, False), (w.clone().requires_grad_(), True)):
        rows = y * 1.0
        out = povs.combine_rows(rows, plan, weights)
        assert any(t is not None and t.shape == y.shape for t in out.grad_fn.saved_tensors) == kept
        if not kept:
            rows.detach().add_(1.0)  # so it may change before the backward pass
        up = _randn(16, 5, seed=2)
        (dy,) = torch.autograd.grad(out, y, up)
        want = torch.zeros(32, 5, device=DEV)
        share = torch.ones(16, 2, device=DEV) if weights is None else weights.detach()
        want[plan.slots.long().reshape(-1)] = (share.unsqueeze(2) * up.unsqueeze(1)).reshape(32, 5)
        assert torch.equal(dy, want)


def test_rows_of_lazily_conjugated_and_negated_tensors():
    """A conjugate or an imaginary part of one is a view whose numbers differ from its bytes."""
    plan = povs.plan_rows(torch.tensor([[1], [0], [1]], dtype=torch.int32, device=DEV), 2)
    z = torch.complex(_randn(3, 4, seed=1), _randn(3, 4, seed=2)).conj()
    assert z.is_conj()
    order = [1, 0, 2]
    assert torch.equal(povs.dispatch_rows(z, plan), z.resolve_conj()[order])
    line = z.imag[:, 0]
    assert line.is_neg()
    assert torch.equal(povs.dispatch_rows(line, plan), line.resolve_neg()[order])
    back = [1, 0, 2]
    assert torch.equal(povs.combine_rows(line, plan), line.resolve_neg()[back])
    column = z.imag[:, :1]
    u = torch.tensor([0.1, 0.2, 0.3], device=DEV)
    assert torch.equal(povs.route(column, 1).weights, torch.ones(3, 1, device=DEV))
    assert torch.equal(povs.route(column, 1, scoring="sigmoid").weights,
                       povs.route(column.resolve_neg(), 1, scoring="sigmoid").weights)
    flat = torch._neg_view(_randn(3, 50, seed=3))
    assert torch.equal(povs.sample(flat, u, top_k=1), povs.sample(flat.resolve_neg(), u, top_k=1))
    assert torch.equal(povs.route(flat, 3).experts, povs.route(flat.resolve_neg(), 3).experts)


@pytest.mark.parametrize("n,groups,top_groups,k", [(248, 31, 9, 8), (240, 30, 4, 8), (240, 3, 2, 5), (8, 1, 1, 8),
                                                   (256, 32, 8, 8), (200, 1, 1, 3)])
@pytest.mark.parametrize("scoring,bias", [("softmax", False), ("sigmoid", True)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_route_of_many_rows_of_every_shape_of_the_tile(dtype, scoring, bias, n, groups, top_groups, k):
    """Rows that one lane, or two to eight, walk, up to the largest tile of shared memory."""
    rows = 9477
    x = _randn(rows, n, seed=n, sharp=1.5, dtype=dtype)
    kw = dict(scoring=scoring, n_groups=groups, top_groups=top_groups)
    if bias:
        kw["bias"] = _randn(n, seed=1, sharp=0.1)
    got = povs.route(x, k, **kw)
    experts, weights = oracle.route(_host(x), k, **{**kw, "bias": _host(kw["bias"]) if bias else None})
    np.testing.assert_array_equal(_host(got.experts), experts)
    np.testing.assert_allclose(_host(got.weights), weights, rtol=_weight_bound(_host(x), n), atol=1e-37)


@pytest.mark.parametrize("renormalize", [False, True])
def test_route_gradient_of_weights_whose_gradients_are_near(renormalize):
    """A softmax over all chosen experts passes on the differences of the weights' gradients alone."""
    x = _randn(60, 4, seed=13)
    x[:, 0] += 5.0
    x = x.requires_grad_()
    experts, weights = povs.route(x, 4, renormalize=renormalize, scale=2.3)
    g = 1.0 + _randn(60, 4, seed=14, sharp=1e-3)
    (dx,) = torch.autograd.grad(weights, x, g)
    want, size = _gradient(_host(x), _host(experts), _host(g), "softmax", renormalize, 2.3)
    assert (np.abs(_host(dx) - want) <= _gradient_bound(size, want, torch.float32, _host(x), 4)).all()
