"""Row operators on the GPU against their definitions in 64 bits (tests/rows_oracle.py).

Tolerances count roundings: one to the output's type is at most ``finfo(t).eps / 2`` relative, one
operation in 32 bits 2^-24 relative.  Whole numbers (ids, experts, slots) are equal.
"""

from __future__ import annotations

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


def _scores(rows: int, width: int, dtype: torch.dtype, seed: int, sharp: float = 2.0) -> torch.Tensor:
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, width, generator=g) * sharp).to(dtype).to(DEV)


def _uniforms(rows: int, seed: int) -> torch.Tensor:
    return torch.rand(rows, generator=torch.Generator().manual_seed(seed)).to(DEV)


# ------------------------------------------------------------------------------------------
# sample
# ------------------------------------------------------------------------------------------


def _sample_wanted(logits, uniforms, **kw):
    x, u = _host(logits), _host(uniforms)
    per_row = {k: _host(v) if isinstance(v, torch.Tensor) else [v] * len(x) for k, v in kw.items()}
    return np.array([oracle.sample_row(x[r], u[r], **{k: v[r].item() if hasattr(v[r], "item") else v[r]
                                                      for k, v in per_row.items()}) for r in range(len(x))])


SETTINGS = [
    {},
    {"temperature": 0.0},
    {"temperature": 0.3},
    {"temperature": 5.0},
    {"top_k": 1},
    {"top_k": 7},
    {"top_k": 100_000},
    {"top_p": 0.0},
    {"top_p": 0.5},
    {"top_p": 0.97},
    {"min_p": 0.1},
    {"min_p": 1.0},
    {"temperature": 0.7, "top_k": 50, "top_p": 0.9, "min_p": 0.02},
    {"temperature": 2.0, "top_k": 3, "top_p": 0.6},
]


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("width", [1, 2, 33, 1000, 4097, 50021])
def test_sample_matches_its_definition(width, dtype, kw):
    rows = 5 if width > 10_000 else 40
    x, u = _scores(rows, width, dtype, seed=width), _uniforms(rows, seed=width + 1)
    got = povs.sample(x, u, **kw)
    assert got.dtype == torch.int64 and got.shape == (rows,)
    np.testing.assert_array_equal(_host(got), _sample_wanted(x, u, **kw))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("width", [3, 1021, 32768, 131071])
def test_sample_settings_of_each_row(width, dtype):
    rows = 30
    g = torch.Generator().manual_seed(width)
    pick = torch.randint(0, 4, (4, rows), generator=g)
    kw = dict(
        temperature=torch.tensor([0.0, 0.5, 1.0, 1.7])[pick[0]].to(DEV),
        top_k=torch.tensor([0, 1, 20, 500], dtype=torch.int32)[pick[1]].to(DEV),
        top_p=torch.tensor([1.0, 0.3, 0.9, 0.99])[pick[2]].to(DEV),
        min_p=torch.tensor([0.0, 0.0, 0.05, 0.5])[pick[3]].to(DEV),
    )
    x, u = _scores(rows, width, dtype, seed=7), _uniforms(rows, seed=8).double()
    np.testing.assert_array_equal(_host(povs.sample(x, u, **kw)), _sample_wanted(x, u, **kw))


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_sample_rows_with_masks(dtype, kw):
    """Rows whose masks (-inf, NaN, the type's lowest value) leave nothing, one id, or ties."""
    width = 2053
    x = _scores(16, width, dtype, seed=3)
    inf, low = float("inf"), torch.finfo(dtype).min
    x[0] = -inf
    x[1] = float("nan")
    x[2] = -inf
    x[2, 1777] = -3.0
    x[3, ::2] = float("nan")
    x[4] = low
    x[5] = low
    x[5, width - 1] = 1.0
    x[6] = 0.5  # every id tied
    x[7] = torch.where(torch.arange(width, device=DEV) % 3 == 0, 1.0, -inf).to(dtype)
    x[8, 100:200] = inf
    x[9] = inf
    x[10] = -0.0
    x[10, 5] = 0.0
    x[11, :1000] = -inf
    x[12] = torch.finfo(dtype).max
    x[13, 0] = torch.finfo(dtype).max
    u = _uniforms(16, seed=4)
    np.testing.assert_array_equal(_host(povs.sample(x, u, **kw)), _sample_wanted(x, u, **kw))


@pytest.mark.parametrize("kw", [{"top_p": 0.9}, {"top_p": 0.999}, {"top_p": 0.6, "min_p": 1e-4}, {"top_k": 5000},
                                {"top_k": 30_000, "top_p": 0.95}, {"min_p": 1e-4}, {"top_p": 0.9, "temperature": 30.0},
                                {"top_p": 0.95, "temperature": 0.01}, {"top_p": 0.5, "temperature": 1e28}], ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows", [3, 40])
def test_sample_wide_nuclei(rows, dtype, kw):
    """Kept sets of thousands of ids: flat scores, scores tied by the thousand, masked runs, few and many
    blocks per row."""
    width = 40_009
    g = torch.Generator().manual_seed(rows)
    x = (torch.randn(rows, width, generator=g) * 0.7).to(dtype).to(DEV)
    x[0] = (x[0] * 2).round() / 2
    x[1, 1000:30_000] = -float("inf")
    x[2] = torch.where(torch.arange(width, device=DEV) < 9000, 3.0, x[2])
    u = _uniforms(rows, seed=11)
    np.testing.assert_array_equal(_host(povs.sample(x, u, **kw)), _sample_wanted(x, u, **kw))


def test_sample_scores_at_the_ends_of_float():
    """Rows of the lowest and highest floats, and temperatures at and beyond both ends."""
    low, high = torch.finfo(torch.float32).min, torch.finfo(torch.float32).max
    width = 3001
    x = torch.full((8, width), low, device=DEV)
    x[1, 7::9] = -float("inf")
    x[2, 3::2] = high
    x[3] = torch.linspace(-1e-30, 1e-30, width, device=DEV)
    x[4] = torch.linspace(low / 2, high / 2, width, device=DEV)
    x[5, :1500] = -float("inf")
    x[5, 2000] = -3.2e38
    x[6] = 1.0
    x[6, 5] = torch.nextafter(torch.tensor(1.0), torch.tensor(2.0))
    u = _uniforms(8, seed=2)
    for temperature in (1e-30, 1e-7, 1.0, 1e10, 1e20):
        for kw in ({}, {"top_p": 0.5}, {"top_k": 50}, {"min_p": 0.3}):
            kw = dict(kw, temperature=temperature)
            np.testing.assert_array_equal(_host(povs.sample(x, u, **kw)), _sample_wanted(x, u, **kw), err_msg=str(kw))


def test_sample_uniforms_at_and_beyond_their_ends():
    x = _scores(6, 301, torch.float32, seed=1)
    x[:, 280:] = -float("inf")
    u = torch.tensor([0.0, 1.0 - 2.0**-24, 1.0, 7.5, -1.0, float("nan")], device=DEV)
    want = [0, 279, 279, 279, 0, 0]
    assert povs.sample(x, u).tolist() == want
    assert povs.sample(x, u.double()).tolist() == want


def test_sample_shares_follow_the_weights():
    """Evenly spaced random numbers draw each id as often as its weight says, up to one per border."""
    n = 20_000
    row = torch.tensor([1.0, -float("inf"), 0.0, 2.0, 1.5, -3.0], device=DEV)
    u = ((torch.arange(n, dtype=torch.float64) + 0.5) / n).to(DEV)
    ids = povs.sample(row.expand(n, -1), u, temperature=0.8)
    w = np.exp(_host(row) / 0.8)
    counts = np.bincount(_host(ids), minlength=6)
    assert np.abs(counts - n * w / w.sum()).max() <= 1


def test_sample_row_strides_and_unaligned_rows():
    base = _scores(9, 1003, torch.bfloat16, seed=2)
    u = _uniforms(9, seed=3)
    for view in (base[:, 1:], base[:, 3:900], base[::2, 7:]):
        np.testing.assert_array_equal(_host(povs.sample(view, u[: len(view)], top_p=0.9, top_k=60)),
                                      _sample_wanted(view, u[: len(view)], top_p=0.9, top_k=60))
    same = base[:1].expand(9, -1)
    np.testing.assert_array_equal(_host(povs.sample(same, u)), _sample_wanted(same, u))


def test_sample_no_rows():
    assert povs.sample(torch.empty(0, 10, device=DEV), torch.empty(0, device=DEV)).shape == (0,)


def test_sample_many_rows_and_wide_rows():
    x, u = _scores(3000, 130, torch.float16, seed=5), _uniforms(3000, seed=6)
    np.testing.assert_array_equal(_host(povs.sample(x, u, top_p=0.8)), _sample_wanted(x, u, top_p=0.8))
    x, u = _scores(2, 1_500_001, torch.float32, seed=7), _uniforms(2, seed=8)
    for kw in ({}, {"top_k": 1000}, {"top_p": 0.95}, {"min_p": 0.01}):
        np.testing.assert_array_equal(_host(povs.sample(x, u, **kw)), _sample_wanted(x, u, **kw))


# ------------------------------------------------------------------------------------------
# route
# ------------------------------------------------------------------------------------------

# (experts, top_k, settings)
ROUTES = [
    (1, 1, {}),
    (2, 2, {"renormalize": True}),
    (8, 2, {"renormalize": True}),
    (31, 5, {"scoring": "sigmoid"}),
    (60, 4, {"bias": True}),
    (64, 6, {"renormalize": True, "scale": 0.5}),
    (128, 8, {}),
    (160, 6, {"n_groups": 8, "top_groups": 3, "group_score": "max", "scale": 16.0}),
    (256, 8, {"scoring": "sigmoid", "bias": True, "n_groups": 8, "top_groups": 4, "renormalize": True, "scale": 2.5}),
    (256, 32, {"scoring": "sigmoid", "n_groups": 32, "top_groups": 5}),
    (12, 3, {"n_groups": 12, "top_groups": 4, "bias": True}),
    (384, 8, {"scoring": "sigmoid", "bias": True, "renormalize": True}),
    (1024, 10, {"bias": True, "n_groups": 4, "top_groups": 2}),
]


def _route_settings(n, kw, seed):
    kw = dict(kw)
    if kw.get("bias"):
        kw["bias"] = (torch.randn(n, generator=torch.Generator().manual_seed(seed)) * 0.1).to(DEV)
    return kw


def _weight_bound(x: np.ndarray, n: int) -> float:
    """Relative error of a weight computed in 32 bits: the rounded difference from the row's highest
    logit (2^-24 of its size, which the exponential turns into a relative error), 4 steps of the
    exponential and the quotient, the sum over n scores and over the chosen ones."""
    finite = x[np.isfinite(x)]
    spread = finite.max() - finite.min() if finite.size else 0.0
    return (spread + n / 32 + 32 + 16) * U32


@pytest.mark.parametrize("n,k,kw", ROUTES, ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows", [1, 77])
def test_route_matches_its_definition(rows, dtype, n, k, kw):
    kw = _route_settings(n, kw, seed=n)
    x = _scores(rows, n, dtype, seed=n + rows, sharp=1.5)
    got = povs.route(x, k, **kw)
    assert got.experts.dtype == torch.int32 and got.weights.dtype == torch.float32
    host = {**kw, "bias": _host(kw["bias"])} if "bias" in kw else kw
    experts, weights = oracle.route(_host(x), k, **host)
    np.testing.assert_array_equal(_host(got.experts), experts)
    np.testing.assert_allclose(_host(got.weights), weights, rtol=_weight_bound(_host(x), n), atol=1e-37)


@pytest.mark.parametrize("kw", [{}, {"renormalize": True}, {"scoring": "sigmoid"}, {"scoring": "sigmoid", "renormalize": True},
                                {"bias": True}, {"n_groups": 4, "top_groups": 2}], ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_route_rows_with_masks_and_ties(dtype, kw):
    n, k = 48, 6
    kw = _route_settings(n, kw, seed=5)
    x = _scores(14, n, dtype, seed=9)
    inf = float("inf")
    x[0] = -inf
    x[1] = -inf
    x[1, 40] = 1.0
    x[2] = 0.25
    x[3, ::2] = -inf
    x[4] = torch.finfo(dtype).min
    x[5, :45] = -inf
    x[6, 3] = float("nan")
    x[7] = float("nan")
    x[8, 9] = inf
    x[9, :] = x[9, 0]
    x[9, 17] += 1
    x[10, 0] = torch.finfo(dtype).max
    x[11, 12:24] = -inf
    host = {**kw, "bias": _host(kw["bias"])} if "bias" in kw else kw
    experts, weights = oracle.route(_host(x), k, **host)
    got = povs.route(x, k, **kw)
    np.testing.assert_array_equal(_host(got.experts), experts)
    np.testing.assert_allclose(_host(got.weights), weights, rtol=64 * U32 + 32 * U32, atol=1e-37)


@pytest.mark.parametrize("n,k,kw", [
    (8, 8, {}),
    (64, 6, {"renormalize": True}),
    (128, 8, {"scoring": "sigmoid"}),
    (128, 1, {"bias": True}),
    (256, 8, {"scoring": "sigmoid", "bias": True, "n_groups": 8, "top_groups": 4, "renormalize": True, "scale": 2.5}),
    (160, 6, {"n_groups": 4, "top_groups": 2, "group_score": "max"}),
    (512, 4, {"scoring": "sigmoid", "n_groups": 32, "top_groups": 9}),
    (384, 7, {"bias": True, "renormalize": True}),
], ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_route_of_many_rows(dtype, n, k, kw):
    """Batches that fill the GPU with one lane per row, the last warp in part, among them masked, tied and
    close rows."""
    rows = 9503
    kw = _route_settings(n, kw, seed=n)
    x = _scores(rows, n, dtype, seed=n, sharp=1.5)
    inf = float("inf")
    x[5] = -inf
    x[40, 1:] = -inf
    x[41, ::2] = -inf
    x[77] = 0.5
    x[78] = x[78, 0]
    x[78, n - 1] += 1
    x[100] = torch.finfo(dtype).min
    x[101, 3] = inf
    x[102, 2] = float("nan")
    x[9502, 0] = torch.finfo(dtype).max
    x[200:260] = (x[200:260] * 4).round() / 4
    x[300] = torch.linspace(-1e-6, 1e-6, n, device=DEV).to(dtype)
    got = povs.route(x, k, **kw)
    host = {**kw, "bias": _host(kw["bias"])} if "bias" in kw else kw
    experts, weights = oracle.route(_host(x), k, **host)
    np.testing.assert_array_equal(_host(got.experts), experts)
    plain = np.ones(rows, bool)
    plain[[5, 40, 41, 100, 101, 102, 9502]] = False
    # As _weight_bound, with a softmax's sum over all n scores by one lane.
    bound = _weight_bound(_host(x)[plain], n) + n * U32
    np.testing.assert_allclose(_host(got.weights), weights, rtol=bound, atol=1e-37)


def test_route_masked_by_bias_and_row_strides():
    n, k = 40, 4
    x = _scores(33, 2 * n, torch.float16, seed=1)[:, 3:3 + n]
    bias = torch.zeros(n, device=DEV)
    bias[5:38] = -float("inf")
    got = povs.route(x, k, bias=bias)
    experts, weights = oracle.route(_host(x), k, bias=_host(bias))
    assert (experts[:, 3] >= 0).all() and set(np.unique(experts)) <= {0, 1, 2, 3, 4, 38, 39}
    np.testing.assert_array_equal(_host(got.experts), experts)
    np.testing.assert_allclose(_host(got.weights), weights, rtol=_weight_bound(_host(x), n))
    same = x[:1].expand(33, -1)
    assert torch.equal(povs.route(same, k).experts[32], povs.route(x[:1], k).experts[0])


def test_route_close_scores_are_told_apart_in_64_bits():
    """Choice scores that differ by less than 32 bits resolve: with a balance bias that undoes the
    scores' differences to within 1e-9, the order is that of the 64-bit sums."""
    n, rows = 64, 50
    x = _scores(rows, n, torch.float32, seed=21, sharp=0.5)
    x[1:] = x[0] + torch.randn(rows - 1, n, device=DEV, generator=torch.Generator(DEV).manual_seed(3)) * 1e-7
    s = np.stack([oracle.scores(r, "sigmoid") for r in _host(x)])
    bias = torch.tensor(0.9 - s[0], dtype=torch.float32, device=DEV)
    got = povs.route(x, 8, scoring="sigmoid", bias=bias)
    experts, _ = oracle.route(_host(x), 8, scoring="sigmoid", bias=_host(bias))
    np.testing.assert_array_equal(_host(got.experts), experts)


GRADIENTS = [(n, k, kw) for n, k, kw in ROUTES if "n_groups" not in kw]


def _gradient_bound(size: np.ndarray, want: np.ndarray, dtype: torch.dtype, x: np.ndarray, n: int) -> np.ndarray:
    """One rounding to the type, and 32-bit arithmetic on terms of the given size: each is a product
    of a score and sums of scores, so three times the relative error of a weight."""
    tiny = {torch.float32: 2.0**-126, torch.bfloat16: 2.0**-126, torch.float16: 2.0**-24}[dtype]
    return torch.finfo(dtype).eps / 2 * np.abs(want) + 3 * _weight_bound(x, n) * size + tiny


@pytest.mark.parametrize("n,k,kw", GRADIENTS, ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_route_gradient_matches_its_formula(dtype, n, k, kw):
    kw = _route_settings(n, kw, seed=n)
    x = _scores(41, n, dtype, seed=n, sharp=1.5).requires_grad_()
    experts, weights = povs.route(x, k, **kw)
    g = torch.randn(41, k, generator=torch.Generator().manual_seed(n)).to(DEV)
    (dx,) = torch.autograd.grad(weights, x, g)
    assert dx.dtype == dtype and dx.shape == x.shape
    want, size = oracle.route_gradient(_host(x), _host(experts), _host(g), kw.get("scoring", "softmax"),
                                       kw.get("renormalize", False), kw.get("scale", 1.0))
    assert (np.abs(_host(dx) - want) <= _gradient_bound(size, want, dtype, _host(x), n)).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_route_gradient_matches_differences(scoring, renormalize):
    """Central differences of the definition in 64 bits, the choices held: truncation (h^2/6 times a
    third derivative of at most 6 |g| scale) and rounding (2^-52 / h) stay below 1e-7 at h = 1e-4."""
    n, k, h, scale = 24, 4, 1e-4, 1.5
    x = _scores(3, n, torch.float32, seed=2, sharp=1.0).requires_grad_()
    experts, weights = povs.route(x, k, scoring=scoring, renormalize=renormalize, scale=scale)
    g = torch.randn(3, k, generator=torch.Generator().manual_seed(4)).to(DEV)
    (dx,) = torch.autograd.grad(weights, x, g)
    base, e, gh = _host(x), _host(experts), _host(g)
    want = np.zeros_like(base)
    for i in range(n):
        step = np.zeros_like(base)
        step[:, i] = h
        up, down = (oracle.weights_of(base + d, e, scoring, renormalize, scale) for d in (step, -step))
        want[:, i] = ((up - down) * gh).sum(1) / (2 * h)
    _, size = oracle.route_gradient(base, e, gh, scoring, renormalize, scale)
    assert (np.abs(_host(dx) - want) <= 3 * _weight_bound(base, n) * size + 1e-6).all()


def test_route_gradient_of_masked_and_padded_rows():
    x = _scores(6, 20, torch.float32, seed=8)
    x[0] = -float("inf")
    x[1, :18] = -float("inf")
    x[2, ::2] = -float("inf")
    for scoring in ("softmax", "sigmoid"):
        for renormalize in (False, True):
            leaf = x.clone().requires_grad_()
            experts, weights = povs.route(leaf, 4, scoring=scoring, renormalize=renormalize)
            (dx,) = torch.autograd.grad(weights.sum(), leaf)  # an expanded gradient
            want, size = oracle.route_gradient(_host(x), _host(experts), np.ones((6, 4)), scoring, renormalize, 1.0)
            assert torch.isfinite(dx).all() and (dx[0] == 0).all() and (dx[x == -float("inf")] == 0).all()
            assert (np.abs(_host(dx) - want) <= _gradient_bound(size, want, torch.float32, _host(x), 20)).all()


# ------------------------------------------------------------------------------------------
# plan, dispatch, combine
# ------------------------------------------------------------------------------------------


def _experts(rows, k, n, seed, padded=0.1, dtype=torch.int32):
    g = np.random.default_rng(seed)
    e = g.integers(0, n, size=(rows, k))
    e[g.random(rows) < padded] = -1
    e[g.random((rows, k)) < padded / 4] = -1
    return torch.from_numpy(e).to(dtype).to(DEV)


@pytest.mark.parametrize("id_dtype", [torch.int32, torch.int64], ids=str)
@pytest.mark.parametrize("rows,k,n", [(0, 3, 5), (1, 1, 1), (13, 6, 64), (1000, 4, 7), (1024, 4, 256), (1025, 4, 3),
                                      (5000, 8, 60), (2053, 2, 4096), (40_000, 8, 256), (70_001, 8, 1),
                                      (300, 40, 1000)])
def test_plan_is_the_stable_order(rows, k, n, id_dtype):
    e = _experts(rows, k, n, seed=rows + k, dtype=id_dtype)
    plan = povs.plan_rows(e, n)
    slots, sources, offsets = oracle.plan(_host(e), n)
    for got, want in zip(plan, (slots, sources, offsets)):
        assert got.dtype == torch.int32
        np.testing.assert_array_equal(_host(got), want)


def test_plan_leaves_out_numbers_outside_the_experts():
    e = torch.tensor([[0, 5], [7, 2**31 - 1], [-1, -(2**31)], [3, 0]], dtype=torch.int32, device=DEV)
    plan = povs.plan_rows(e, 5)
    assert plan.slots.tolist() == [[0, -1], [-1, -1], [-1, -1], [2, 1]]
    assert plan.sources.tolist() == [0, 7, 6, -1, -1, -1, -1, -1]
    assert plan.offsets.tolist() == [0, 2, 2, 2, 3, 3]
    big = e.long() + torch.tensor([[0, 2**32]], device=DEV)
    assert povs.plan_rows(big, 5).offsets.tolist() == [0, 1, 1, 1, 2, 2]


def test_plan_of_padding_only():
    plan = povs.plan_rows(torch.full((9000, 2), -1, dtype=torch.int32, device=DEV), 17)
    assert (plan.slots == -1).all() and (plan.sources == -1).all() and (plan.offsets == 0).all()
    x = torch.randn(9000, 5, device=DEV)
    assert (povs.dispatch_rows(x, plan) == 0).all()
    assert (povs.combine_rows(torch.randn(18000, 5, device=DEV), plan) == 0).all()


SHAPES = [(1, 1, (1,)), (13, 6, (2048,)), (50, 2, (7,)), (33, 3, (129,)), (200, 4, (64,)), (17, 9, (3, 5, 4)),
          (9, 1, (4096,)), (6, 40, (24,)), (100, 8, (1000,)), (5, 2, (1023,))]


@pytest.mark.parametrize("dtype", [*DTYPES, torch.uint8, torch.int64, torch.bool], ids=str)
@pytest.mark.parametrize("rows,k,shape", SHAPES)
def test_dispatch_moves_rows(rows, k, shape, dtype):
    g = torch.Generator().manual_seed(rows)
    x = torch.randint(-100, 100, (rows, *shape), generator=g).to(dtype).to(DEV)
    plan = povs.plan_rows(_experts(rows, k, 11, seed=rows), 11)
    got = povs.dispatch_rows(x, plan)
    assert got.shape == (rows * k, *shape) and got.dtype == dtype
    raw = x.cpu().to(torch.float64).numpy()
    np.testing.assert_array_equal(got.cpu().to(torch.float64).numpy(), oracle.dispatch(raw, _host(plan.slots)))


def _one_rounding(want: np.ndarray, dtype: torch.dtype) -> np.ndarray:
    return torch.finfo(dtype).eps / 2 * np.abs(want) + torch.finfo(dtype).smallest_normal


@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,k,shape", SHAPES)
def test_combine_sums_rows(rows, k, shape, dtype, weighted):
    g = torch.Generator().manual_seed(rows)
    y = torch.randn(rows * k, *shape, generator=g).to(dtype).to(DEV)
    w = torch.randn(rows, k, generator=g).to(DEV) if weighted else None
    plan = povs.plan_rows(_experts(rows, k, 11, seed=rows), 11)
    got = povs.combine_rows(y, plan, w)
    want, size = oracle.combine(_host(y), _host(plan.slots), None if w is None else _host(w))
    assert got.shape == (rows, *shape) and got.dtype == dtype
    # k products and sums in 32 bits, one rounding to the type.
    assert (np.abs(_host(got) - want) <= _one_rounding(want, dtype) + (k + 1) * U32 * size).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,k,shape", SHAPES)
def test_dispatch_and_combine_gradients(rows, k, shape, dtype):
    g = torch.Generator().manual_seed(rows)
    plan = povs.plan_rows(_experts(rows, k, 11, seed=rows), 11)
    slots = _host(plan.slots)
    x = torch.randn(rows, *shape, generator=g).to(dtype).to(DEV).requires_grad_()
    up = torch.randn(rows * k, *shape, generator=g).to(dtype).to(DEV)
    (dx,) = torch.autograd.grad(povs.dispatch_rows(x, plan), x, up)
    want, size = oracle.combine(_host(up), slots, None)
    assert dx.dtype == dtype and (np.abs(_host(dx) - want) <= _one_rounding(want, dtype) + k * U32 * size).all()

    y = torch.randn(rows * k, *shape, generator=g).to(dtype).to(DEV).requires_grad_()
    w = torch.randn(rows, k, generator=g).to(DEV).requires_grad_()
    up = torch.randn(rows, *shape, generator=g).to(dtype).to(DEV)
    dy, dw = torch.autograd.grad(povs.combine_rows(y, plan, w), (y, w), up)
    hy, hw, hu = _host(y), _host(w), _host(up)
    here = slots >= 0
    want_y = np.zeros_like(hy)
    want_w, size_w = np.zeros(slots.shape), np.zeros(slots.shape)
    for r, j in zip(*np.nonzero(here)):
        want_y[slots[r, j]] = hu[r] * hw[r, j]
        want_w[r, j] = (hu[r] * hy[slots[r, j]]).sum()
        size_w[r, j] = np.abs(hu[r] * hy[slots[r, j]]).sum()
    assert (np.abs(_host(dy) - want_y) <= _one_rounding(want_y, dtype) + U32 * np.abs(want_y)).all()
    assert (_host(dw)[~here] == 0).all()
    # Sums of `width` products in 32 bits, in any order.
    assert (np.abs(_host(dw) - want_w) <= (np.prod(shape) + 1) * U32 * size_w).all()
    # One gradient alone, and the sums' gradient through a broadcast.
    (only,) = torch.autograd.grad(povs.combine_rows(y.detach(), plan, w), w, up)
    assert torch.equal(only, dw)
    (only,) = torch.autograd.grad(povs.combine_rows(y, plan, w.detach()), y, up)
    assert torch.equal(only, dy)
    (ones,) = torch.autograd.grad(povs.combine_rows(y, plan).sum(), y)
    assert torch.equal(ones, torch.zeros_like(ones).index_fill_(0, plan.slots[plan.slots >= 0].long(), 1.0))


def test_dispatch_and_combine_row_strides():
    plan = povs.plan_rows(_experts(64, 3, 9, seed=1), 9)
    wide = torch.randn(64, 100, device=DEV).to(torch.bfloat16)
    for view in (wide[:, 8:72], wide[:, 1:50], wide[:, 4:8]):
        assert torch.equal(povs.dispatch_rows(view, plan), povs.dispatch_rows(view.contiguous(), plan))
    assert torch.equal(povs.dispatch_rows(wide[:1].expand(64, -1), plan), povs.dispatch_rows(wide[:1].repeat(64, 1), plan))
    wide = torch.randn(192, 100, device=DEV).to(torch.bfloat16)
    w = torch.rand(64, 3, device=DEV)
    for view in (wide[:, 8:72], wide[:, 1:50]):
        assert torch.equal(povs.combine_rows(view, plan, w), povs.combine_rows(view.contiguous(), plan, w))
        leaf = view.detach().requires_grad_()
        flat = view.contiguous().requires_grad_()
        wl = w.clone().requires_grad_()
        a = torch.autograd.grad(povs.combine_rows(leaf, plan, wl).float().pow(2).sum(), (leaf, wl))
        b = torch.autograd.grad(povs.combine_rows(flat, plan, wl).float().pow(2).sum(), (flat, wl))
        assert torch.equal(a[0], b[0])
        # A weight's gradient sums the same products in another order where rows are read in other
        # pieces: each sum is within (width + 1) 2^-24 of its terms' size of the exact one.
        here = plan.slots >= 0
        terms = (2 * povs.combine_rows(flat.detach(), plan, w).double().unsqueeze(1)
                 * flat.detach().double()[plan.slots.clamp(min=0).long()]).abs().sum(2)
        bound = torch.where(here, 2 * (view.shape[1] + 1) * U32 * terms, 0.0)
        assert ((a[1].double() - b[1].double()).abs() <= bound).all()
    line = torch.arange(128, device=DEV)[::2]
    assert torch.equal(povs.dispatch_rows(line, plan), povs.dispatch_rows(line.contiguous(), plan))


def test_plans_with_slots_out_of_range_touch_nothing_outside():
    """A plan made by hand may hold places that do not exist: they are left out."""
    slots = torch.tensor([[0, 4], [2**31 - 1, 1], [-7, 3]], dtype=torch.int32, device=DEV)
    plan = povs.RowPlan(slots, torch.empty(0, dtype=torch.int32, device=DEV),
                        torch.tensor([0, 2**31 - 1], dtype=torch.int32, device=DEV))
    x = torch.arange(6.0, device=DEV).reshape(3, 2)
    got = povs.dispatch_rows(x, plan)
    assert torch.equal(got[[0, 1, 3, 4]], x[[0, 1, 2, 0]])
    y = torch.arange(12.0, device=DEV).reshape(6, 2)
    assert torch.equal(povs.combine_rows(y, plan), torch.stack([y[0] + y[4], y[1], y[3]]))


def test_rows_past_32_bit_offsets():
    """More than 2^32 bytes of rows: 70 000 rows of 33 KiB to two places each."""
    rows, width, k = 70_000, 33 * 1024, 2
    free, _ = torch.cuda.mem_get_info()
    if free < 16 << 30:
        pytest.skip("needs 16 GiB of device memory")
    x = torch.randint(0, 256, (rows, width), dtype=torch.uint8, device=DEV)
    plan = povs.plan_rows(_experts(rows, k, 5, seed=3, padded=0.0), 5)
    out = povs.dispatch_rows(x, plan)
    at = torch.tensor([0, 1, rows // 2, rows - 1], device=DEV)
    for j in range(k):
        places = plan.slots[at, j].long()
        here = places >= 0
        assert torch.equal(out[places[here]], x[at[here]])
    del x
    y = out.view(torch.bfloat16)
    got = povs.combine_rows(y, plan)
    for r in at.tolist():
        here = [s for s in plan.slots[r].tolist() if s >= 0]
        want = sum(y[s].float() for s in here) if here else torch.zeros(width // 2, device=DEV)
        assert torch.equal(got[r].nan_to_num(), want.to(torch.bfloat16).nan_to_num())


# ------------------------------------------------------------------------------------------
# Together, on streams and in graphs.
# ------------------------------------------------------------------------------------------


def _layer(x, gate, w1, head, u):
    """Rows routed to experts, each expert's product, combined, an id drawn for every row."""
    experts, weights = povs.route(x @ gate, 2, renormalize=True)
    plan = povs.plan_rows(experts, w1.shape[0])
    rows = povs.dispatch_rows(x, plan)
    which = torch.searchsorted(plan.offsets, torch.arange(rows.shape[0], device=DEV, dtype=torch.int32), right=True) - 1
    which = which.clamp(max=w1.shape[0] - 1)
    y = torch.bmm(rows.unsqueeze(1), w1[which]).squeeze(1)
    out = povs.combine_rows(y, plan, weights)
    return experts, out, povs.sample((out @ head).detach(), u, top_k=20, top_p=0.95)


def test_a_layer_of_experts_and_its_gradients():
    g = torch.Generator().manual_seed(0)
    n, d, e, v = 37, 24, 6, 101

    def randn(*s):
        return torch.randn(*s, generator=g, dtype=torch.float32).to(DEV)

    x, gate, w1, head = randn(n, d).requires_grad_(), randn(d, e).requires_grad_(), randn(e, d, d).requires_grad_(), randn(d, v)
    u = torch.rand(n, generator=g).to(DEV)
    experts, out, ids = _layer(x, gate, w1, head, u)
    up = randn(n, d)
    got = torch.autograd.grad(out, (x, gate, w1), up)
    xd, gd, wd = (t.detach().double().requires_grad_() for t in (x, gate, w1))
    s = torch.softmax(xd @ gd, 1)
    w, best = s.topk(2, dim=1)
    assert torch.equal(best.int(), experts)
    w = w / w.sum(1, keepdim=True)
    want_out = sum(torch.bmm(xd.unsqueeze(1), wd[best[:, j]]).squeeze(1) * w[:, j:j + 1] for j in range(2))
    want = torch.autograd.grad(want_out, (xd, gd, wd), up.double())
    # Products of length 24 in 32 bits (about 24 roundings on values of order 24), then sums over up
    # to 37 rows: 1e-4 of the largest value is an order of magnitude above.
    for a, b in zip((out, *got), (want_out, *want)):
        assert (a.double() - b).abs().max() <= 1e-4 * b.abs().max()
    np.testing.assert_array_equal(_host(ids), _sample_wanted(out.detach() @ head, u, top_k=20, top_p=0.95))


def test_captured_and_replayed_with_new_inputs():
    rows, n, k, d, v = 50, 16, 2, 40, 5000
    x, logits, scores = torch.randn(rows, d, device=DEV), torch.randn(rows, n, device=DEV), torch.randn(rows, v, device=DEV)
    u = torch.rand(rows, device=DEV)

    def step():
        experts, weights = povs.route(logits, k)
        plan = povs.plan_rows(experts, n)
        return experts, povs.combine_rows(povs.dispatch_rows(x, plan), plan, weights), povs.sample(scores, u, top_p=0.9)

    graphs = []
    for _ in range(2):  # two graphs of the same calls, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    for i in range(4):
        for t in (x, logits, scores):
            t.normal_()
        u.uniform_()
        want = step()
        graph, outs = graphs[i % 2]
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_captured_training_step():
    rows, n, k, d = 64, 8, 2, 32
    x, logits = torch.randn(rows, d, device=DEV), torch.randn(rows, n, device=DEV)

    def step():
        xl, ll = x.detach().requires_grad_(), logits.detach().requires_grad_()
        experts, weights = povs.route(ll, k, renormalize=True)
        plan = povs.plan_rows(experts, n)
        out = povs.combine_rows(povs.dispatch_rows(xl, plan) * 2.0, plan, weights)
        return torch.autograd.grad((out * out).sum(), (xl, ll))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(2):
        x.normal_()
        logits.normal_()
        want = step()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_calls_on_two_streams_at_once():
    rows, n, d, v = 4000, 64, 256, 32000
    data = [(torch.randn(rows, n, device=DEV), torch.randn(rows, d, device=DEV), torch.randn(64, v, device=DEV),
             torch.rand(64, device=DEV)) for _ in range(2)]

    def step(logits, x, scores, u):
        experts, weights = povs.route(logits, 4)
        plan = povs.plan_rows(experts, n)
        return povs.combine_rows(povs.dispatch_rows(x, plan), plan, weights), povs.sample(scores, u, top_k=100, top_p=0.9)

    want = [step(*d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(*data[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))


def test_refusals():
    x, u = torch.zeros(4, 8, device=DEV), torch.zeros(4, device=DEV)
    plan = povs.plan_rows(torch.zeros(4, 2, dtype=torch.int32, device=DEV), 3)
    rows = torch.zeros(8, 5, device=DEV)
    for call in (
        lambda: povs.sample(x.double(), u), lambda: povs.sample(x, u.half()), lambda: povs.sample(x, u.cpu()),
        lambda: povs.sample(x, u, temperature=u.double()), lambda: povs.sample(x, u, top_k=u),
        lambda: povs.route(x.double(), 2), lambda: povs.route(x, 2, bias=torch.zeros(8, device=DEV).half()),
        lambda: povs.route(x, 2, bias=torch.zeros(8)), lambda: povs.plan_rows(x, 3),
        lambda: povs.dispatch_rows(x.cpu(), plan), lambda: povs.dispatch_rows(x, plan._replace(slots=plan.slots.long())),
        lambda: povs.combine_rows(rows.double(), plan), lambda: povs.combine_rows(rows, plan, torch.zeros(4, 2, device=DEV).half()),
        lambda: povs.dispatch_rows(x.double().requires_grad_(), plan),
    ):
        with pytest.raises(TypeError):
            call()
    for call in (
        lambda: povs.sample(x.t(), u), lambda: povs.sample(x[0], u), lambda: povs.sample(x, u[:3]),
        lambda: povs.sample(x, u, temperature=-1.0), lambda: povs.sample(x, u, temperature=float("nan")),
        lambda: povs.sample(x, u, top_k=-1), lambda: povs.sample(x, u, top_p=1.5), lambda: povs.sample(x, u, min_p=-0.5),
        lambda: povs.sample(x, u, top_p=u[:2]), lambda: povs.sample(x[:, :0], u),
        lambda: povs.route(x.t(), 2), lambda: povs.route(x, 0), lambda: povs.route(x, 9), lambda: povs.route(x, 2, scoring="relu"),
        lambda: povs.route(x, 2, n_groups=3), lambda: povs.route(x, 2, n_groups=4, top_groups=5),
        lambda: povs.route(x, 3, n_groups=4, top_groups=1), lambda: povs.route(x, 2, group_score="mean"),
        lambda: povs.route(x, 2, scale=float("inf")), lambda: povs.route(x, 2, bias=torch.zeros(7, device=DEV)),
        lambda: povs.route(torch.zeros(2, 1025, device=DEV), 2), lambda: povs.plan_rows(plan.slots.t(), 3),
        lambda: povs.plan_rows(plan.slots, 0), lambda: povs.plan_rows(plan.slots, 4097), lambda: povs.plan_rows(plan.slots[0], 3),
        lambda: povs.dispatch_rows(x[:3], plan), lambda: povs.dispatch_rows(x.t()[:4], plan),
        lambda: povs.combine_rows(rows[:7], plan), lambda: povs.combine_rows(rows, plan, torch.zeros(4, 3, device=DEV)),
        lambda: povs.combine_rows(rows, plan, torch.zeros(2, 4, device=DEV).t()),
    ):
        with pytest.raises(AssertionError):
            call()


def test_row_operators_take_numpy_numbers_and_huge_top_k():
    x, u = _scores(4, 50, torch.float32, seed=1), _uniforms(4, seed=2)
    kw = dict(temperature=np.float32(0.5), top_k=np.int64(7), top_p=np.float32(0.5), min_p=np.float64(0.25))
    np.testing.assert_array_equal(_host(povs.sample(x, u, **kw)), _sample_wanted(x, u, **{k: float(v) if k != "top_k" else 7 for k, v in kw.items()}))
    assert torch.equal(povs.sample(x, u, top_k=2**70), povs.sample(x, u))
    assert torch.equal(povs.route(x, np.int32(3), scale=np.float32(2)).weights, povs.route(x, 3, scale=2.0).weights)


def test_gradients_refuse_a_second_order():
    plan = povs.plan_rows(_experts(8, 2, 4, seed=1), 4)
    for make in (lambda t: povs.route(t, 2).weights, lambda t: povs.dispatch_rows(t, plan)):
        x = torch.randn(8, 6, device=DEV).requires_grad_()
        with pytest.raises(RuntimeError, match="once differentiable"):
            torch.autograd.grad(make(x).sum(), x, create_graph=True)
    y = torch.randn(16, 6, device=DEV).requires_grad_()
    with pytest.raises(RuntimeError, match="once differentiable"):
        torch.autograd.grad(povs.combine_rows(y, plan).sum(), y, create_graph=True)


def test_same_inputs_same_bits():
    x, u = _scores(20, 100_000, torch.bfloat16, seed=1), _uniforms(20, seed=2)
    logits = _scores(5000, 128, torch.float32, seed=3)
    runs = [(povs.sample(x, u, top_p=0.9), *povs.route(logits, 8, scoring="sigmoid")) for _ in range(3)]
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))
