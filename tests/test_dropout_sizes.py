"""Dropout on either side of the sizes where its loads and stores change: a call's bytes, and its result's, beside the 256 MB of the
last-level cache."""
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "awesome-cute_amd"))
sys.path.insert(0, os.path.join(ROOT, "tests"))
import _masks  # noqa: E402
import feedforward  # noqa: E402

gpu = pytest.mark.gpu
CACHE = 256 << 20


@gpu
@pytest.mark.parametrize("type", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("matrices", [1, 2, 3])
@pytest.mark.parametrize("more", [-8, 0, 1, 8, 1027])
def test_results_beside_the_caches_size(matrices, more, type):
    """matrices: those of a call (its result alone, or with the operand, or with the residual too) that fill the cache."""
    size = torch.finfo(type).bits // 8
    count = CACHE // (size * matrices) + more
    gen = torch.Generator(device="cuda").manual_seed(count)
    x, residual = (torch.randn(count, device="cuda", generator=gen).to(type) for _ in range(2))
    few = 4096 + 13
    for r in (None, residual):
        y = feedforward.dropout(x, 0.25, 9, site=4, residual=r)
        # the first elements are those of a small call: places are counted from the start
        assert torch.equal(y[:few], feedforward.dropout(x[:few], 0.25, 9, site=4, residual=None if r is None else r[:few]))
        # the last ones, by the generator
        first = (count - 64) // 8 * 8
        words = [_masks.philox((g, 0, 4, 0), (9, 0), 7) for g in range(first // 8, (count + 7) // 8)]
        keep = torch.tensor([w[e // 2] >> 16 * (e % 2) & 0xffff >= 16384 for w in words for e in range(8)], device="cuda")
        keep = keep[:count - first]
        zero = torch.zeros((), dtype=torch.double, device="cuda")
        # in 64 bits: a factor of 4/3, off by 2^-24, its product's rounding, the addition's, and half a step of the result
        v = torch.where(keep, x[first:].double() * (4 / 3), zero)
        want = v if r is None else v + r[first:].double()
        bound = 2.0 ** -22 * (v.abs() + (0 if r is None else r[first:].double().abs())) + torch.finfo(type).eps / 2 * want.abs() * 1.02
        assert ((y[first:].double() - want).abs() <= bound + 2.0 ** -25).all()
        # ... and as many are dropped as should be, six deviations wide
        dropped = (y == (0 if r is None else r)).float().mean(dtype=torch.double).item()
        assert abs(dropped - 0.25) < 6 * (0.25 * 0.75 / count) ** 0.5 + 2.0 ** -10
        del y
