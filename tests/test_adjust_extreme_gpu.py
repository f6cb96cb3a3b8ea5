"""Repetition penalties at the ends of what a number holds: the quotient and its reciprocal
pass 64 bits there, the result is the rounding of the exact one (infinite past the type)."""

from __future__ import annotations

import pytest
import torch

import test_adjust_gpu as adjust

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("r", [5e-324, 1e-320, 5.5e-309, 5.6e-309, 1e-300, 1e-271, 1e-269, 1e-100,
                               1e-40, 1e40, 1e100, 1e307, 1.7e308])
def test_repetition_penalties_far_from_one(r, dtype):
    info = torch.finfo(dtype)
    x = torch.tensor([info.max, info.min, info.smallest_normal, -info.smallest_normal, 0.0, -0.0,
                      1.0, -1.0, 3e-30, -3e-30, 7e20, -7e20, float("inf"), float("-inf"),
                      float("nan"), 12.5]).to(dtype)
    x = x.repeat(2, 1, 40)[:, :, :637].contiguous()
    prompt = torch.arange(600).expand(2, 600).contiguous()
    output = torch.arange(500, 640).expand(2, 140).contiguous()
    adjust._check(x, prompt=prompt, output=output, r=r)
    adjust._check(x, prompt=prompt, output=output, r=r, f=0.5, p=-0.25)
