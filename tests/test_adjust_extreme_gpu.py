"""Repetition penalties at the ends of what a number holds: the quotient and its reciprocal
pass 64 bits there, the result is the rounding of the exact one (infinite past the type). And
every pattern of bits, NaN's too, beside masked elements: what nothing touches keeps its bits."""

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


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("dtype,bits", [(F32, torch.int32), (BF, torch.int16)])
def test_bits_beside_masked_elements(dtype, bits, inplace):
    g = torch.Generator().manual_seed(2)
    if dtype == BF:
        x = torch.arange(-2 ** 15, 2 ** 15).to(bits)
    else:
        odd = torch.tensor([0x7f800001, 0x7fbfffff, 0x7fc00123, 1, 0x7fffff, 0x800000])
        x = torch.cat([torch.randint(-2 ** 31, 2 ** 31, (60001,), generator=g), odd,
                       odd - 2 ** 31]).to(bits)
    x = x[torch.randperm(x.numel(), generator=g)].view(dtype).expand(1, 3, -1).contiguous()
    v = x.shape[2]
    drafts = torch.full((1, 2), -1)
    allowed = torch.randint(-2 ** 31, 2 ** 31, (1, 3, -(-v // 32)), generator=g).to(torch.int32)
    at = torch.arange(v)
    keep = ((allowed.long()[..., at // 32] >> (at % 32)) & 1).bool()
    got = adjust._run(x.to(adjust.DEV), inplace, drafts=drafts, allowed=allowed).cpu()
    assert torch.equal(got.view(bits)[keep], x.view(bits)[keep])
    assert bool((got[~keep] == float("-inf")).all())
