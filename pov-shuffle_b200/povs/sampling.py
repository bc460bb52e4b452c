"""Drawing ids from scores on the GPU (addition to the reference API).

Where ``numpy.random.Generator`` has ``choice`` beside the ``shuffle`` that ``povs.shuffle`` replaces,
this module draws one id per row of scores.  The random numbers are given by the caller, as
``apply_randomness`` has its offsets and permutations given, so a draw can be repeated.
"""

from __future__ import annotations

import math

import torch

from . import _native


def sample(
    logits: torch.Tensor,
    uniforms: torch.Tensor,
    temperature: float | torch.Tensor = 1.0,
    top_k: int | torch.Tensor = 0,
    top_p: float | torch.Tensor = 1.0,
    min_p: float | torch.Tensor = 0.0,
) -> torch.Tensor:
    """Draw one id per row: an int64 tensor (rows,), asynchronous on the current stream.

    With the weights ``w = exp((x - max x) / temperature)`` of a row's scores ``x`` and the ids ordered by
    descending score (equal scores by the lowest id), ``top_k`` keeps the first ids, ``top_p`` keeps of
    those the ids before which less than that share of their weight lies (the first always), and
    ``min_p`` keeps of those the ids with at least that weight (the highest score has weight 1 and
    always stays).  The result is the lowest id at which the kept weights, summed in id order, exceed
    the row's uniform number times their sum.  NaN and -inf scores are never drawn; where scores are
    +inf, one of them is; a row without any number above -inf gives -1.  Weights and sums have 64
    bits and are good to 2^-40 of the row's sum (``top_p``'s border, where it keeps thousands of ids of a row of
    ``2**n``, to ``2**(2 * n - 63)`` at worst); the same inputs give the same ids on every run.  Temperatures
    above 1e28 count as 1e28, those below 1e-36 as 1e-36.

    :param logits: CUDA tensor (rows, width) of float32, bfloat16 or float16; ids contiguous, any row stride.
    :param uniforms: (rows,) float32 or float64 in [0, 1), contiguous, on the same device.
    :param temperature: 0 takes the highest score.  Like the other three, a number for all rows or a
        contiguous tensor (rows,): float32 (``top_k``: int32).  Tensor values are not checked: a temperature
        not above 0 takes the highest score, a ``top_k`` not above 0 and a ``top_p`` of 1 or more keep every id.
    :param top_k: Number of ids kept, 0 for all.
    :param top_p: Share of the weight kept, in [0, 1]; 1 for all.
    :param min_p: Lowest weight kept relative to the highest, in [0, 1]; 0 for all.
    """
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise TypeError("sample takes a CUDA tensor of scores")
    _native.score_dtype(logits)
    logits = _native.plain(logits)
    assert logits.dim() == 2, f"logits must have shape (rows, width), got {tuple(logits.shape)}"
    rows, width = logits.shape
    assert width >= 1, "logits must have at least one id per row"
    assert width == 1 or logits.stride(1) == 1, "ids of a row must be contiguous"
    uniforms = _per_row("uniforms", uniforms, logits, (torch.float32, torch.float64))
    given = {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p}
    for name, value in given.items():
        if isinstance(value, torch.Tensor):
            given[name] = _per_row(name, value, logits, (torch.int32 if name == "top_k" else torch.float32,))
    temperature, top_k, top_p, min_p = given.values()
    if not isinstance(temperature, torch.Tensor):
        assert temperature >= 0 and math.isfinite(temperature), f"temperature ({temperature}) must be finite and at least 0"
    if not isinstance(top_k, torch.Tensor):
        assert top_k >= 0, f"top_k ({top_k}) must be at least 0"
        top_k = min(int(top_k), width)
    if not isinstance(top_p, torch.Tensor):
        assert 0 <= top_p <= 1, f"top_p ({top_p}) must be in [0, 1]"
    if not isinstance(min_p, torch.Tensor):
        assert 0 <= min_p <= 1, f"min_p ({min_p}) must be in [0, 1]"
    return _native.sample(logits, uniforms, temperature, top_k, top_p, min_p)


def _per_row(name: str, value: torch.Tensor, logits: torch.Tensor, dtypes: tuple) -> torch.Tensor:
    if not isinstance(value, torch.Tensor) or value.device != logits.device:
        raise TypeError(f"{name} must be a tensor on the device of logits ({logits.device})")
    if value.dtype not in dtypes:
        raise TypeError(f"{name} must have dtype {' or '.join(map(str, dtypes))}, got {value.dtype}")
    assert value.shape == (logits.shape[0],), f"{name} must have shape ({logits.shape[0]},), got {tuple(value.shape)}"
    assert value.is_contiguous(), f"{name} must be contiguous"
    return _native.plain(value)
