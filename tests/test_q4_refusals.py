"""What the 4-bit cache's entry points refuse, checked without a GPU: every
check of the C ABI runs before any CUDA call, and the Python wrappers refuse
tensors before they reach it."""

import ctypes

import pytest
import torch

from aegaeon_b200 import _lib, q4_cache

P = 0x7F0000000000  # a 16-byte aligned address that is never touched


def write(kvx, **kw):
    a = dict(key=P, value=P, dtype=0, tokens=1, kt=1024, kh=128, vt=1024, vh=128, slots=P, kp=P,
             vp=P, stride=8704, blocks=4, heads=8, block=16, dim=128, stream=None)
    a.update(kw)
    return kvx.kvx_q4_write(*a.values())


def read(kvx, **kw):
    a = dict(kp=P, vp=P, stride=8704, blocks=4, heads=8, block=16, dim=128, slots=P, tokens=1,
             key=P, value=P, dtype=0, kt=1024, kh=128, vt=1024, vh=128, stream=None)
    a.update(kw)
    return kvx.kvx_q4_read(*a.values())


def attend(kvx, **kw):
    a = dict(query=P, qt=4096, qh=128, out=P, ot=4096, oh=128, lse=None, dtype=0, tokens=2,
             num_heads=32, kp=P, vp=P, stride=8704, blocks=4, heads=8, block=16, dim=128,
             tables=P, table_stride=4, width=4, lens=P, starts=None, batch=2, scale=0.1, window=0,
             sinks=0, work=P, work_bytes=1 << 40, stream=None)
    a.update(kw)
    return kvx.kvx_q4_attention(*a.values())


CACHE = [
    dict(dim=96), dict(dim=0), dict(block=0), dict(block=24), dict(block=8192), dict(heads=0),
    dict(heads=1025, stride=1 << 30), dict(blocks=-1), dict(kp=None), dict(vp=None),
    dict(kp=P + 8), dict(stride=8712), dict(stride=8688), dict(stride=-16),
]


@pytest.mark.parametrize("bad", CACHE + [
    dict(dtype=3), dict(tokens=-1), dict(key=None), dict(slots=None), dict(key=P + 1),
    dict(dtype=2, value=P + 2)])
def test_write_and_read_refuse(kvx, bad):
    assert write(kvx, **bad) == _lib.KVX_ERR_INVALID_ARGUMENT
    assert kvx.kvx_last_error()
    assert read(kvx, **bad) == _lib.KVX_ERR_INVALID_ARGUMENT


def test_nothing_to_do_is_no_error(kvx):
    assert write(kvx, tokens=0, key=None, value=None, slots=None) == 0
    assert read(kvx, tokens=0, key=None, value=None, slots=None) == 0
    assert attend(kvx, tokens=0, query=None, out=None) == 0
    assert attend(kvx, batch=0, lens=None, tables=None) == 0


@pytest.mark.parametrize("bad", CACHE + [
    dict(dtype=2), dict(tokens=-1), dict(batch=-1), dict(width=-1), dict(num_heads=0),
    dict(num_heads=12), dict(window=-1), dict(sinks=-1), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(query=None), dict(out=None), dict(lens=None),
    dict(tables=None), dict(query=P + 1), dict(work=P + 4), dict(width=1 << 27),
    dict(tokens=1 << 28, batch=1)])
def test_attention_refuses(kvx, bad):
    assert attend(kvx, **bad) == _lib.KVX_ERR_INVALID_ARGUMENT
    assert kvx.kvx_last_error()


def test_attention_refuses_uneven_queries(kvx):
    assert attend(kvx, tokens=3) == _lib.KVX_ERR_LENGTH_MISMATCH


def test_workspace_query_refuses(kvx):
    n = ctypes.c_uint64()
    assert kvx.kvx_q4_attention_workspace(100, 8, ctypes.byref(n)) == _lib.KVX_ERR_INVALID_ARGUMENT
    assert kvx.kvx_q4_attention_workspace(128, 8, None) == _lib.KVX_ERR_INVALID_ARGUMENT


def test_sizes():
    assert q4_cache.head_bytes(16, 128) == 16 * 68
    assert q4_cache.page_bytes(32, 8, 64) == 8 * 32 * 36
    k, v = q4_cache.allocate(3, 16, 2, 256, device="cpu")
    assert k.shape == v.shape == (3, 2, 16 * 132) and k.dtype is torch.uint8 and not k.any()
    for bad in ((16, 96), (8, 128), (24, 128), (8192, 64)):
        with pytest.raises(ValueError):
            q4_cache.head_bytes(*bad)


def test_wrappers_refuse_before_the_library():
    k, v = q4_cache.allocate(4, 16, 2, 128, device="cpu")
    x = torch.zeros(5, 2, 128, dtype=torch.bfloat16)
    slots = torch.arange(5)
    with pytest.raises(ValueError, match="CUDA"):
        q4_cache.write(x, x, k, v, slots)
    with pytest.raises(ValueError, match="CUDA"):
        q4_cache.read(k, v, slots, head_dim=128)
    with pytest.raises(ValueError, match="CUDA"):
        q4_cache.attention(x, k, v, torch.zeros(5, 1, dtype=torch.int32),
                           torch.zeros(5, dtype=torch.int32))
    with pytest.raises(TypeError, match="uint8"):
        q4_cache.write(x, x, k.view(torch.int8), v, slots)
    with pytest.raises(ValueError, match="one shape"):
        q4_cache.write(x, x, k, v[:3], slots)
    with pytest.raises(ValueError, match="head_dim"):
        q4_cache.write(x[..., :96], x[..., :96], k, v, slots)
    with pytest.raises(ValueError, match="tokens, kv_heads"):
        q4_cache.write(x[0], x[0], k, v, slots)
