"""GPU tests of the 4-bit cache where its numbers and its memory are easily got
wrong: rows at the ends of the value range, value scales far apart, weights and
queries of extreme size, and arguments that share memory.

Expected values come from the definition in 64 bits (q4_oracle)."""

import math

import pytest
import torch

import q4_oracle
from aegaeon_b200 import _lib, q4_cache

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def _status(cuda):
    """Each test starts and, unless it clears the word itself, ends with no
    device error."""
    _lib.device_status(0, reset=True)
    yield
    assert _lib.device_status(0, reset=True) == 0


def randn(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


# ---- rows at the ends of the range ----------------------------------------------------


def rows_beyond_fp16(dim):
    """fp32 rows that lie close to the largest fp16 and have values beyond it."""
    rows = []
    for low, high in ((65500.0, 70000.0), (65040.004, 70000.0), (65490.0, 1e6), (65300.0, 1e6),
                      (65503.9, 3e38), (65504.0, 65505.0), (65024.0, 66000.0), (7e4, 3e5)):
        x = torch.full((dim,), low)
        x[dim // 2] = high
        rows.append(x)
    g = torch.Generator().manual_seed(1)
    for _ in range(56):
        x = 65024 + 480 * torch.rand(dim, generator=g) ** (1 + 3 * torch.rand(1, generator=g))
        x[torch.randint(dim, (3,), generator=g)] = 65504 * (1 + torch.rand(3, generator=g))
        rows.append(x)
    return torch.stack(rows)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_codes_of_clamped_rows_follow_the_definition(dim):
    """A value beyond +-65504 counts as that value, not only in the row's ends."""
    rows = rows_beyond_fp16(dim).cuda()[:, None]
    block = 16
    kp, vp = q4_cache.allocate(-(-rows.shape[0] // block), block, 1, dim)
    slots = torch.arange(rows.shape[0], device="cuda")
    q4_cache.write(rows, -rows, kp, vp, slots)
    for pages, x in ((kp, rows), (vp, -rows)):
        codes, scale, zero = (t[:, 0].flatten(0, 1)[:rows.shape[0]] for t in q4_oracle.split(pages, dim))
        want = q4_oracle.quantise(x[:, 0])
        assert torch.equal(scale, want[1][:, 0]) and torch.equal(zero, want[2][:, 0])
        assert torch.equal(codes, want[0])
