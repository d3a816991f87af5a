"""Shared checks of the training-step operators' tests: results in 64 bits to compare with,
and how far off a result may be.

Tolerances, on the 2-norm of the difference over that of the exact result:

* an output rounded to bfloat16 once: every element is off by at most 2^-9 of itself, plus
  float32 arithmetic before the rounding (below): 2^-8;
* float32: each value takes a few roundings of 2^-24 and a sum of n terms adds at most
  about log2(n) + n / threads of them along any path, each of its partial sum: 2e-6 for
  rows (n <= 16384), 1e-5 for sums over rows, whose terms cancel.
"""

from __future__ import annotations

import torch

BF16 = 2.0 ** -8
F32_ROW = 2e-6
F32_SUM = 1e-5


def off(got: torch.Tensor, exact: torch.Tensor) -> float:
    assert got.shape == exact.shape, (got.shape, exact.shape)
    got, exact = got.detach().double().cpu(), exact.detach().double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(exact))
    finite = torch.isfinite(exact)
    assert torch.equal(got[~finite].nan_to_num(7.0), exact[~finite].nan_to_num(7.0))
    norm = exact[finite].norm().item()
    diff = (got[finite] - exact[finite]).norm().item()
    return diff / norm if norm else diff


def check(got: torch.Tensor, exact: torch.Tensor, f32: float, what: str = "") -> None:
    bound = BF16 if got.dtype == torch.bfloat16 else f32
    d = off(got, exact)
    assert d <= bound, f"{what}: off by {d:.3e}, at most {bound:.3e}"


def leaf(t):
    return t.detach().double().requires_grad_(True) if isinstance(t, torch.Tensor) else t


def randn(gen, *shape, dtype=torch.float32, scale=1.0):
    """Seeded on the host: the same input on every machine."""
    return (torch.randn(*shape, generator=gen) * scale).to(dtype)
