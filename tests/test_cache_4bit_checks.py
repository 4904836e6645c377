"""Checks of the 4-bit cache's arguments that need no GPU."""

import random

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from aegaeon_b200 import _lib, q4_cache
from test_q4_refusals import P, attend, read, write


def places(t):
    """The elements of the storage that a tensor names."""
    at = torch.zeros((), dtype=torch.int64) + t.storage_offset()
    for n, s in zip(t.shape, t.stride()):
        at = at[..., None] + torch.arange(n) * s
    return at.flatten().tolist()


def test_overlap_of_strided_views():
    """Any two views of one storage, against a list of their elements."""
    overlap = _lib.q4().overlap
    rng = random.Random(5)
    base = torch.zeros(100000, dtype=torch.int16)
    shared = apart = 0
    for _ in range(4000):
        views = []
        for _ in range(2):
            dims = rng.randint(1, 3)
            size = [rng.randint(1, 5) for _ in range(dims)]
            stride, inner = [], 1
            for n in reversed(size):  # mostly nested, as views of one tensor are
                stride.append(rng.choice([inner, inner + rng.randint(0, 6), rng.randint(0, 40)]))
                inner = max(1, stride[-1] * n)
            stride.reverse()
            views.append(base.as_strided(size, stride, rng.randint(0, 300)))
        want = not set(places(views[0])).isdisjoint(places(views[1]))
        assert overlap(*views) == want, [(v.shape, v.stride(), v.storage_offset()) for v in views]
        shared, apart = shared + want, apart + (not want)
    assert shared > 500 and apart > 500


def test_overlap_of_the_views_that_callers_have():
    overlap = _lib.q4().overlap
    qkv = torch.zeros(100, 48, 128, dtype=torch.float16)
    q, k, v = qkv[:, :32], qkv[:, 32:40], qkv[:, 40:]
    assert overlap(q, qkv[:, :32]) and overlap(q, qkv[:, 31:40]) and overlap(qkv, v)
    assert not overlap(q, k) and not overlap(k, v) and not overlap(q, torch.zeros(5))
    pages = torch.zeros(50, 4, 2, 8, 1088, dtype=torch.uint8)  # blocks, layers, K and V
    for i in range(4):
        for j in range(4):
            for a in range(2):
                for b in range(2):
                    assert overlap(pages[:, i, a], pages[:, j, b]) == ((i, a) == (j, b))
    assert overlap(pages[:, 1], pages[7]) and not overlap(pages[:7], pages[7:])
    empty = qkv[:0]
    assert not overlap(empty, qkv) and not overlap(qkv, empty)
    long = torch.zeros(1, dtype=torch.float16).expand(100000, 7, 128)  # one element, many names
    assert overlap(long, long) and not overlap(long, qkv)


def test_forward_mode_gradients_are_refused():
    """A dual tensor's tangent would be lost without a word."""
    kp, vp = q4_cache.allocate(2, 16, 2, 128, device="cpu")
    x, slots = torch.zeros(3, 2, 128), torch.arange(3)
    half, tables, lens = x.half(), torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    with forward_ad.dual_level():
        dual, dual_half = forward_ad.make_dual(x, x + 1), forward_ad.make_dual(half, half + 1)
        view = dual[:, :, :]
        for call in (lambda: q4_cache.write(dual, x, kp, vp, slots),
                     lambda: q4_cache.write(x, view, kp, vp, slots),
                     lambda: q4_cache.attention(dual_half, kp, vp, tables, lens)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with torch.no_grad():  # turns reverse mode off, not this one
            with pytest.raises(RuntimeError, match="forward-mode"):
                q4_cache.write(dual, x, kp, vp, slots)
    with pytest.raises(ValueError, match="CUDA"):  # the level is over
        q4_cache.write(dual, x, kp, vp, slots)


@pytest.mark.parametrize("bad", [
    dict(tables=P + 2), dict(lens=P + 1), dict(starts=P + 2, tokens=3), dict(lse=P + 3),
    dict(width=1 << 60), dict(width=(1 << 60) + 4), dict(num_heads=1 << 62, tokens=4, batch=1),
    dict(num_heads=8 << 33), dict(tokens=1 << 62, batch=1), dict(batch=1 << 62, starts=P),
    dict(stride=1 << 62)])
def test_attention_refuses_what_would_wrap_or_misalign(kvx, bad):
    """Pointers that a kernel would load 4 bytes from, and sizes whose products pass 64 bits."""
    assert attend(kvx, **bad) == _lib.KVX_ERR_INVALID_ARGUMENT
    assert kvx.kvx_last_error()


@pytest.mark.parametrize("bad", [dict(slots=P + 4), dict(tokens=1 << 62), dict(tokens=1 << 31),
                                 dict(stride=1 << 62)])
def test_write_and_read_refuse_what_would_wrap_or_misalign(kvx, bad):
    assert write(kvx, **bad) == _lib.KVX_ERR_INVALID_ARGUMENT
    assert read(kvx, **bad) == _lib.KVX_ERR_INVALID_ARGUMENT
