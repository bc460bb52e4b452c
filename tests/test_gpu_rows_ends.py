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
