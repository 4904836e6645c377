"""GPU tests of the 4-bit paged cache against its definition in 64 bits.

Codes, scales and zeros are compared exactly, and so are rows read back.
Attention is held to the bound that q4_oracle.attention derives for each
element."""

import math

import pytest
import torch

import q4_oracle
from aegaeon_b200 import _lib, ops, q4_cache, swapper

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def _status(cuda):
    """Each test starts and, unless it clears the word itself, ends with no
    device error."""
    _lib.device_status(0, reset=True)
    yield
    assert _lib.device_status(0, reset=True) == 0


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, dtype, seed):
    return torch.randn(shape, generator=gen(seed), device="cuda").to(dtype)


def expected_pages(pages, rows, slots, dim):
    """Pages (CPU) after rows were written into slots."""
    pages = pages.cpu().clone()
    block = pages.shape[2] // (dim // 2 + 4)
    codes, scale, zero = q4_oracle.quantise(rows)
    packed = codes[..., 0::2] | (codes[..., 1::2] << 4)
    params = torch.cat([scale, zero], -1)
    half = block * dim // 2
    to_codes = pages[..., :half].unflatten(-1, (block, dim // 2))
    to_params = pages[..., half:].view(torch.float16).unflatten(-1, (block, 2))
    for i, s in enumerate(slots.tolist()):
        if s >= 0:
            to_codes[s // block, :, s % block] = packed[i]
            to_params[s // block, :, s % block] = params[i]
    return pages


def assert_pages(got, want, dim):
    """Bytes equal, but that a NaN is any NaN."""
    g, w = q4_oracle.split(got, dim), q4_oracle.split(want, dim)
    assert torch.equal(g[0], w[0])
    for a, b in zip(g[1:], w[1:]):
        assert torch.equal(a.isnan(), b.isnan())
        assert torch.equal(a.nan_to_num(), b.nan_to_num())


def noise(shape, seed):
    """Pages that were used before: any bytes."""
    return torch.randint(0, 256, shape, generator=gen(seed), device="cuda", dtype=torch.uint8)


@pytest.mark.parametrize("tokens,heads,dim,block", [
    (1, 1, 128, 16), (1, 8, 64, 16), (7, 3, 128, 16), (33, 2, 256, 32), (130, 5, 64, 48),
    (257, 4, 128, 128), (64, 1, 256, 16)])
@pytest.mark.parametrize("dtype", DTYPES + [torch.float32])
def test_write_and_read(tokens, heads, dim, block, dtype):
    blocks = tokens // block + 3
    shape = (blocks, heads, q4_cache.head_bytes(block, dim))
    kp, vp = noise(shape, 1), noise(shape, 2)
    key, value = randn((tokens, heads, dim), dtype, 3), 3 + randn((tokens, heads, dim), dtype, 4)
    slots = torch.randperm(blocks * block, generator=gen(5), device="cuda")[:tokens]
    slots[tokens // 2:tokens // 2 + tokens // 5] = -1
    want_k, want_v = expected_pages(kp, key, slots, dim), expected_pages(vp, value, slots, dim)
    q4_cache.write(key, value, kp, vp, slots)
    assert_pages(kp, want_k, dim)
    assert_pages(vp, want_v, dim)
    for out_type in DTYPES + [torch.float32]:
        got = q4_cache.read(kp, vp, slots, head_dim=dim, dtype=out_type)
        for g, pages in zip(got, (kp, vp)):
            x = q4_oracle.values(pages, dim).float()
            at = slots.cpu().clamp(min=0)
            want = torch.where((slots.cpu() >= 0)[:, None, None], x[at // block, :, at % block],
                               torch.zeros(()))
            assert torch.equal(g.cpu(), want.to(out_type))


def special_rows(dtype, dim):
    rows = []
    top = torch.finfo(dtype).max
    rows.append(torch.zeros(dim))
    rows.append(torch.full((dim,), 1.5))
    rows.append(torch.arange(dim) % 16)                      # scale 1: no rounding
    rows.append((torch.arange(dim) % 31) / 2.0)              # every second value on a border
    rows.append(((torch.arange(dim) % 31) - 7) * 1.5)        # borders, scale no power of two
    rows.append(((torch.arange(dim) % 46) + 1000.0) * 0.25)  # an offset far above the range
    rows.append(torch.linspace(-1, 1, dim) * 1e-6)           # scale near fp16's smallest
    rows.append(torch.linspace(0, 1, dim) * 1e-8)            # scale below it: all codes 0
    rows.append(torch.linspace(-1, 1, dim) * min(top, 3e5))  # beyond fp16 for bf16 and fp32
    for bad in (math.nan, math.inf, -math.inf):
        x = torch.linspace(-1, 1, dim)
        x[dim // 3] = bad
        rows.append(x)
    x = torch.full((dim,), -0.0)
    x[5] = 1e-3
    rows.append(x)
    return torch.stack(rows).to(dtype)[:, None]


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES + [torch.float32])
def test_write_special_rows(dtype, dim):
    rows = special_rows(dtype, dim).cuda()
    kp, vp = q4_cache.allocate(2, 16, 1, dim)
    slots = torch.arange(rows.shape[0], device="cuda") + 3
    q4_cache.write(rows, -rows, kp, vp, slots)
    assert_pages(kp, expected_pages(torch.zeros_like(kp), rows, slots, dim), dim)
    assert_pages(vp, expected_pages(torch.zeros_like(vp), -rows, slots, dim), dim)
    key, _ = q4_cache.read(kp, vp, slots, head_dim=dim, dtype=torch.float32)
    finite = torch.isfinite(rows.float()).all(-1)
    assert torch.equal(key.isnan().all(-1), ~finite) and torch.equal(key.isnan().any(-1), ~finite)


def test_codes_on_borders_follow_the_definition():
    """Values spread over few steps, where quotients meet borders often."""
    g = gen(11)
    rows = torch.randint(-64, 65, (4096, 2, 128), generator=g, device="cuda").to(torch.bfloat16)
    rows *= torch.tensor([0.125, 3.0], device="cuda", dtype=torch.bfloat16)[None, :, None]
    kp, vp = q4_cache.allocate(256, 16, 2, 128)
    slots = torch.arange(4096, device="cuda")
    q4_cache.write(rows, rows, kp, vp, slots)
    assert_pages(kp, expected_pages(torch.zeros_like(kp), rows, slots, 128), 128)


@pytest.mark.parametrize("offset,pad", [(0, 8), (1, 3), (8, 0), (4, 0)])
def test_strided_rows_and_pages(offset, pad):
    """Rows inside a fused projection, at any alignment, and K and V pages
    interleaved in one tensor."""
    tokens, heads, dim, block = 45, 3, 128, 16
    wide = randn((tokens, 2 * heads, dim + pad), torch.bfloat16, 6)
    flat = torch.cat([wide.reshape(-1), torch.zeros(16, dtype=torch.bfloat16, device="cuda")])
    view = flat[offset:offset + wide.numel()].view(tokens, 2 * heads, dim + pad)[..., :dim]
    key, value = view[:, :heads], view[:, heads:]
    pages = noise((9, 2, heads, q4_cache.head_bytes(block, dim)), 7)
    before = pages.clone()
    kp, vp = pages[:, 0], pages[:, 1]
    slots = torch.randperm(9 * block, generator=gen(8), device="cuda")[:tokens]
    want = expected_pages(kp, key, slots, dim), expected_pages(vp, value, slots, dim)
    q4_cache.write(key, value, kp, vp, slots)
    assert torch.equal(kp.cpu(), want[0]) and torch.equal(vp.cpu(), want[1])
    assert not torch.equal(before, pages)
    out = torch.full((2, tokens, heads, dim + pad + 1), 7.0, dtype=torch.float16, device="cuda")
    view = out[..., 1:dim + 1] if offset else out[..., :dim]
    a, b = q4_cache.read(kp, vp, slots, head_dim=dim, out=(view[0], view[1]))
    plain = q4_cache.read(kp, vp, slots, head_dim=dim, dtype=torch.float16)
    assert torch.equal(a, plain[0]) and torch.equal(b, plain[1])
    rest = out[..., dim + 1:] if offset else out[..., dim:]
    assert (rest == 7).all() and (not offset or (out[..., 0] == 7).all())


def test_slots_outside_the_cache_are_skipped_and_reported():
    kp, vp = noise((4, 2, q4_cache.head_bytes(16, 128)), 1), noise((4, 2, 16 * 68), 2)
    rows = randn((5, 2, 128), torch.float16, 3)
    slots = torch.tensor([3, 64, 2 ** 40, -5, 63], device="cuda")
    ok = torch.tensor([3, -1, -1, -1, 63], device="cuda")
    want = expected_pages(kp, rows, ok, 128)
    q4_cache.write(rows, rows, kp, vp, slots)
    assert _lib.device_status(0, reset=True) == _lib.KVX_ERR_BLOCK_ID
    assert torch.equal(kp.cpu(), want)
    a, _ = q4_cache.read(kp, vp, slots, head_dim=128)
    assert _lib.device_status(0, reset=True) == _lib.KVX_ERR_BLOCK_ID
    b, _ = q4_cache.read(kp, vp, ok, head_dim=128)
    assert torch.equal(a, b) and not a[1:4].any()


# ---- attention --------------------------------------------------------------------


def make_cache(lens, heads, dim, block, seed, spare=2, width=None, garbage=True):
    """Pages of sequences of the given lengths and their block tables.  Bytes
    that belong to no token are anything, NaN patterns among them."""
    need = [-(-n // block) for n in lens]
    blocks = sum(need) + spare
    shape = (blocks, heads, q4_cache.head_bytes(block, dim))
    kp, vp = noise(shape, seed), noise(shape, seed + 1)
    if garbage:
        for p in (kp, vp):
            p[:, :, block * dim // 2:] = 0xFF  # every scale and zero NaN
    order = torch.randperm(blocks, generator=gen(seed + 2), device="cuda").to(torch.int32)
    tables = torch.full((len(lens), width or max(1, max(need, default=1))), -7, device="cuda",
                        dtype=torch.int32)
    at, slots = 0, []
    for i, n in enumerate(need):
        tables[i, :n] = order[at:at + n]
        j = torch.arange(lens[i], device="cuda")
        slots.append(order[at:at + n][j // block].long() * block + j % block if n else j)
        at += n
    slots = torch.cat(slots) if slots else torch.zeros(0, dtype=torch.int64, device="cuda")
    key, value = randn((len(slots), heads, dim), torch.float16, seed + 3), \
        randn((len(slots), heads, dim), torch.float16, seed + 4)
    value = value + 0.5 * randn((1, heads, dim), torch.float16, seed + 5)
    if len(slots):
        q4_cache.write(key, value, kp, vp, slots)
    return kp, vp, tables, torch.tensor(lens, device="cuda", dtype=torch.int32), slots


def check(query, kp, vp, tables, lens, starts=None, **kw):
    got = q4_cache.attention(query, kp, vp, tables, lens, query_starts=starts, return_lse=True, **kw)
    kw.pop("out", None)
    compare(got, q4_oracle.attention(query, kp, vp, tables, lens, starts, **kw), starts)
    return got


def compare(got, want, starts=None):
    out, lse, out_bound, lse_bound = want
    real = slice(None)
    if starts is not None:
        real = slice(int(starts[0]), int(starts[-1]))
    g, gl = got[0][real].double().cpu(), got[1][real].double().cpu()
    off = (g - out[real]).abs()
    assert torch.isfinite(g).all()
    assert (off <= out_bound[real]).all(), f"off by {(off / out_bound[real].clamp(min=1e-30)).max()} bounds"
    none = torch.isinf(lse[real])
    assert torch.equal(none, torch.isinf(gl)) and (gl[none] < 0).all()
    assert (g[none] == 0).all()
    assert ((gl - lse[real]).abs()[~none] <= lse_bound[real][~none]).all()


LENGTHS = [[1], [16], [17, 1, 0, 31], [33, 64, 250], [255, 257, 0, 511, 2], [700, 1, 1100]]


@pytest.mark.parametrize("lens", LENGTHS)
@pytest.mark.parametrize("heads,kv_heads,dim,block", [
    (4, 4, 128, 16), (8, 2, 64, 32), (7, 1, 128, 48), (16, 2, 256, 16), (12, 1, 128, 16),
    (32, 1, 64, 16), (40, 1, 128, 128), (20, 1, 256, 64)])
def test_decode(lens, heads, kv_heads, dim, block):
    kp, vp, tables, lengths, _ = make_cache(lens, kv_heads, dim, block, 20)
    for dtype in DTYPES:
        check(randn((len(lens), heads, dim), dtype, 30), kp, vp, tables, lengths)


@pytest.mark.parametrize("queries", [2, 3, 5, 9])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (20, 0), (64, 4), (33, 17), (500, 500)])
def test_several_queries_and_windows(queries, window, sinks):
    lens = [queries, 1, 0, 18, 130, 517]
    kp, vp, tables, lengths, _ = make_cache(lens, 2, 128, 16, 40)
    query = randn((len(lens) * queries, 6, 128), torch.bfloat16, 41)
    check(query, kp, vp, tables, lengths, window=window, sinks=sinks)


@pytest.mark.parametrize("dim,group,block", [(64, 4, 32), (128, 7, 16), (128, 1, 64), (256, 2, 16)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (48, 4)])
def test_pieces_of_prompts(dim, group, block, window, sinks):
    """Ragged query rows: whole prompts, pieces behind a prefix, a sequence
    without queries, more queries than tokens, and rows behind the last."""
    lens = [70, 300, 40, 0, 129, 5]
    counts = [70, 37, 0, 0, 1, 9]
    kp, vp, tables, lengths, _ = make_cache(lens, 2, dim, block, 50)
    starts = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], device="cuda",
                          dtype=torch.int32)
    tokens = sum(counts) + 6
    query = randn((tokens, 2 * group, dim), torch.float16, 51)
    out = torch.full_like(query, 9.0)
    check(query, kp, vp, tables, lengths, starts, window=window, sinks=sinks, out=out)
    assert (out[-6:] == 9).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,block,counts,lens", [
    (32, 16, 128, 16, [340], [340]),                    # a whole prompt
    (32, 16, 64, 32, [129, 0, 215], [500, 77, 215]),    # behind a prefix, none, whole
    (28, 4, 128, 16, [350, 1, 64, 400], [363, 129, 70, 401]),
    (16, 16, 128, 128, [640], [1000]),
    (64, 8, 64, 48, [160, 5], [161, 3]),                # more queries than tokens
])
@pytest.mark.parametrize("window,sinks", [(None, 0), (100, 4)])
def test_many_rows(dtype, heads, kv_heads, dim, block, counts, lens, window, sinks):
    """Enough rows for the tensor-core kernel (tiles of 128 rows for half the SMs)."""
    assert sum(counts) * (heads // kv_heads) // 128 * kv_heads >= 74
    kp, vp, tables, lengths, _ = make_cache(lens, kv_heads, dim, block, 55)
    starts = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], device="cuda",
                          dtype=torch.int32)
    query = randn((sum(counts) + 3, heads, dim), dtype, 56)
    out = torch.full_like(query, 9.0)
    check(query, kp, vp, tables, lengths, starts, window=window, sinks=sinks, out=out)
    assert (out[-3:] == 9).all()


def test_many_rows_alike_and_strided():
    """The same number of rows for every sequence, query and out inside wider
    tensors, blocks that are not there, and the same result twice."""
    kp, vp, tables, lengths, _ = make_cache([333, 0, 150], 8, 128, 16, 57)
    wide = randn((3 * 110, 40, 136), torch.bfloat16, 58)
    for q in (wide[:, 4:36, :128], wide[:, 4:36, 5:133]):
        want = check(q, kp, vp, tables, lengths)
        out = torch.full((330, 32, 137), 5.0, dtype=torch.bfloat16, device="cuda")
        got = q4_cache.attention(q, kp, vp, tables, lengths, out=out[..., 1:129])
        assert torch.equal(got, want[0])
        assert (out[..., 0] == 5).all() and (out[..., 129:] == 5).all()
    q = wide[:, 4:36, :128]
    want = q4_cache.attention(q, kp, vp, tables, lengths)
    assert torch.equal(want, q4_cache.attention(q, kp, vp, tables, lengths))
    tables[0, 3] = -1
    got = q4_cache.attention(q, kp, vp, tables, lengths)
    assert _lib.device_status(0, reset=True) == _lib.KVX_ERR_BLOCK_ID
    assert torch.isfinite(got).all() and not torch.equal(got[:110], want[:110])
    assert torch.equal(got[110:], want[110:])


def test_many_rows_scales_and_nan():
    lens = [260]
    kp, vp, tables, lengths, slots = make_cache(lens, 16, 128, 16, 59)
    base = randn((170, 64, 128), torch.bfloat16, 60)
    for factor in (1e-30, 40.0, 0.0):
        check(base * factor, kp, vp, tables, lengths)
    check(base, kp, vp, tables, lengths, scale=-0.3)
    key = randn((260, 16, 128), torch.float32, 62)
    value = randn((260, 16, 128), torch.float32, 63)
    grow = torch.exp2(torch.linspace(-18, 13, 260, device="cuda"))[:, None, None]
    for factor in (grow, grow.flip(0), torch.zeros_like(grow)):
        q4_cache.write(key, value * factor, kp, vp, slots)
        check(base, kp, vp, tables, lengths)
    bad = torch.full((1, 16, 128), math.nan, device="cuda")
    fine = torch.ones_like(bad)
    for k, v in ((bad, fine), (fine, bad)):
        q4_cache.write(k, v, kp, vp, slots[200:201])
        got = q4_cache.attention(base, kp, vp, tables, lengths)
        assert torch.isfinite(got[:110]).all() and got[110:].isnan().all()


def test_lengths_that_the_shares_cut():
    """Long enough that many CTAs share a head, at lengths around their borders."""
    for n in (4095, 4096, 4097, 9000):
        kp, vp, tables, lengths, _ = make_cache([n], 1, 128, 16, 60)
        check(randn((1, 7, 128), torch.bfloat16, 61), kp, vp, tables, lengths)


@pytest.mark.parametrize("batch", [129, 700])
def test_more_sequences_than_threads(batch):
    """A thread of the planning looks at several sequences; lengths from nothing up."""
    lens = [(7 * i) % 90 for i in range(batch)]
    lens[batch // 2] = 2000
    kp, vp, tables, lengths, _ = make_cache(lens, 2, 64, 16, 65)
    check(randn((batch, 4, 64), torch.float16, 66), kp, vp, tables, lengths)
    counts = [min(n, i % 3) for i, n in enumerate(lens)]
    starts = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], device="cuda",
                          dtype=torch.int32)
    check(randn((sum(counts), 4, 64), torch.bfloat16, 67), kp, vp, tables, lengths, starts,
          window=30, sinks=2)


def test_many_rows_of_many_sequences():
    lens = [(11 * i) % 60 + 1 for i in range(1100)]
    counts = [min(n, 20) for n in lens]
    assert sum(counts) * 2 // 128 >= 74
    kp, vp, tables, lengths, _ = make_cache(lens, 1, 64, 16, 68)
    starts = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], device="cuda",
                          dtype=torch.int32)
    check(randn((sum(counts), 2, 64), torch.float16, 69), kp, vp, tables, lengths, starts)


def test_scales_and_ranges():
    """Queries of any range, scores far apart, values of small and large scale."""
    lens = [200, 64]
    kp, vp, tables, lengths, slots = make_cache(lens, 1, 128, 16, 70)
    base = randn((2, 4, 128), torch.bfloat16, 71)
    check(base * 1e-30, kp, vp, tables, lengths)
    check(base * 40, kp, vp, tables, lengths)
    check(base * 1e30, kp, vp, tables, lengths, scale=1e-30)
    check(base, kp, vp, tables, lengths, scale=-0.3)
    check(base * 0, kp, vp, tables, lengths)
    key = randn((len(slots), 1, 128), torch.float32, 72)
    value = randn((len(slots), 1, 128), torch.float32, 73)
    grow = torch.exp2(torch.linspace(-18, 13, len(slots), device="cuda"))[:, None, None]
    for factor in (grow, grow.flip(0), torch.zeros_like(grow)):
        q4_cache.write(key, value * factor, kp, vp, slots)
        check(base, kp, vp, tables, lengths)


def test_nan_stays_with_the_rows_that_see_it():
    lens = [90]
    kp, vp, tables, lengths, slots = make_cache(lens, 1, 128, 16, 80)
    bad = torch.full((1, 1, 128), math.nan, device="cuda")
    good = randn((1, 1, 128), torch.float32, 81)
    for key, value in ((bad, good), (good, bad)):
        q4_cache.write(key, value, kp, vp, slots[-2:-1])
        got, lse = q4_cache.attention(randn((4, 2, 128), torch.float16, 82), kp, vp, tables, lengths,
                                      return_lse=True)
        assert torch.isfinite(got[:2]).all() and torch.isfinite(lse[:2]).all()
        assert got[2:].isnan().all()
    q4_cache.write(bad, bad, kp, vp, slots[:1])  # only the windows that reach it see it
    got = q4_cache.attention(randn((1, 2, 128), torch.float16, 82), kp, vp, tables, lengths, window=1)
    assert torch.isfinite(got).all()
    got = q4_cache.attention(randn((1, 2, 128), torch.float16, 82), kp, vp, tables, lengths, window=1,
                             sinks=1)
    assert got.isnan().all()


def test_bad_blocks_and_lengths_are_skipped_and_reported():
    kp, vp, tables, lengths, _ = make_cache([100, 100], 1, 128, 16, 90)
    query = randn((2, 4, 128), torch.bfloat16, 91)
    want = q4_cache.attention(query, kp, vp, tables, lengths)
    for bad in (-1, kp.shape[0], 2 ** 31 - 1):
        t = tables.clone()
        t[1, 3] = bad
        got = q4_cache.attention(query, kp, vp, t, lengths)
        assert _lib.device_status(0, reset=True) == _lib.KVX_ERR_BLOCK_ID
        assert torch.equal(got[0], want[0]) and torch.isfinite(got).all()
        assert not torch.equal(got[1], want[1])
    got = q4_cache.attention(query, kp, vp, tables[:, :5].contiguous(), lengths)
    assert _lib.device_status(0, reset=True) == _lib.KVX_ERR_EXTENT
    short = torch.full_like(lengths, 80)
    assert torch.equal(got, q4_cache.attention(query, kp, vp, tables, short))
    negative = torch.tensor([100, -3], dtype=torch.int32, device="cuda")
    got = q4_cache.attention(query, kp, vp, tables, negative)
    assert torch.equal(got[0], want[0]) and not got[1].any()
    starts = torch.tensor([0, 1, 9], dtype=torch.int32, device="cuda")  # behind the query's end
    got = q4_cache.attention(query, kp, vp, tables, lengths, query_starts=starts)
    assert torch.isfinite(got).all()


def test_strided_arguments():
    kp, vp, tables, lengths, _ = make_cache([77, 30], 2, 128, 16, 100, width=9)
    both = torch.stack([kp, vp], 1)
    wide = randn((2, 14, 131), torch.bfloat16, 101)
    for view in (wide[:, 2:10, :128], wide[:, 2:10, 3:]):
        want = q4_cache.attention(view.contiguous(), kp, vp, tables, lengths)
        out = torch.full((2, 8, 133), 5.0, dtype=torch.bfloat16, device="cuda")
        got = q4_cache.attention(view, both[:, 0], both[:, 1], tables[:, :6], lengths,
                                 out=out[..., 1:129])
        assert torch.equal(got, want)
        assert (out[..., 0] == 5).all() and (out[..., 129:] == 5).all()


def test_same_result_each_time():
    kp, vp, tables, lengths, _ = make_cache([3000, 40, 1700], 2, 128, 16, 110)
    query = randn((3, 8, 128), torch.float16, 111)
    first = q4_cache.attention(query, kp, vp, tables, lengths, return_lse=True)
    for _ in range(5):
        again = q4_cache.attention(query, kp, vp, tables, lengths, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_offsets_beyond_32_bits():
    """A cache of more than 4 GB for each tensor."""
    heads, dim, block = 32, 128, 16
    page = q4_cache.page_bytes(block, heads, dim)
    blocks = 2 ** 32 // page + 40
    kp = torch.zeros((blocks, heads, q4_cache.head_bytes(block, dim)), dtype=torch.uint8, device="cuda")
    vp = torch.zeros_like(kp)
    n = 100
    ids = torch.tensor([blocks - 1, 3, blocks - 30, blocks // 2 + 7, blocks - 2, 0, blocks - 9],
                       device="cuda")
    slots = (ids[:, None] * block + torch.arange(block, device="cuda")).reshape(-1)[:n].contiguous()
    key, value = randn((n, heads, dim), torch.bfloat16, 120), randn((n, heads, dim), torch.bfloat16, 121)
    q4_cache.write(key, value, kp, vp, slots)
    small_k, small_v = kp[ids].contiguous(), vp[ids].contiguous()
    near = torch.arange(n, device="cuda")
    a, b = q4_cache.read(kp, vp, slots, head_dim=dim), q4_cache.read(small_k, small_v, near, head_dim=dim)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and a[0].any()
    query = randn((1, heads, dim), torch.bfloat16, 122)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    x = q4_cache.attention(query, kp, vp, ids[None].int(), lens)
    y = q4_cache.attention(query, small_k, small_v, torch.arange(7, device="cuda")[None].int(), lens)
    assert torch.equal(x, y)


def test_other_stream_and_captured_graphs():
    """Calls on a stream of their own, and two graphs captured over the same
    tensors and replayed in turn and side by side with changed lengths."""
    kp, vp, tables, lengths, slots = make_cache([400, 90], 2, 128, 16, 130)
    query = randn((2, 8, 128), torch.bfloat16, 131)
    key, value = randn((2, 2, 128), torch.bfloat16, 132), randn((2, 2, 128), torch.bfloat16, 133)
    turn = torch.stack([slots[399], slots[-1]])

    def step():
        q4_cache.write(key, value, kp, vp, turn)
        return q4_cache.attention(query, kp, vp, tables, lengths)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert torch.equal(got, want)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for n in ([400, 90], [1, 33], [250, 0]):
        lengths.copy_(torch.tensor(n, dtype=torch.int32))
        expect = step()
        for o in outs:
            o.fill_(7)
        torch.cuda.synchronize()
        graphs[0].replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], expect) and torch.equal(outs[1], expect)


def test_first_call_of_a_kind_inside_a_capture():
    """A call needs nothing outside the capture, not even a kernel's first (run alone,
    this test is the first use of head_dim 256 with more than 8 rows)."""
    kp, vp, tables, lengths, _ = make_cache([300, 40], 1, 256, 32, 135)
    query = randn((2, 11, 256), torch.float16, 136)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = q4_cache.attention(query, kp, vp, tables, lengths)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, q4_cache.attention(query, kp, vp, tables, lengths))


def test_many_heads_of_one_kv_head():
    """128 query heads on one kv head: single tokens take the kernel of many rows
    where there are sequences enough, the other one where there are not."""
    for batch in (80, 3):
        lens = [(37 * i) % 300 + 1 for i in range(batch)]
        kp, vp, tables, lengths, _ = make_cache(lens, 1, 64, 16, 137)
        check(randn((batch, 128, 64), torch.bfloat16, 138), kp, vp, tables, lengths)


def test_nothing_to_do():
    kp, vp = q4_cache.allocate(2, 16, 2, 128)
    none = torch.zeros((0, 2, 128), dtype=torch.bfloat16, device="cuda")
    slots = torch.zeros(0, dtype=torch.int64, device="cuda")
    q4_cache.write(none, none, kp, vp, slots)
    assert q4_cache.read(kp, vp, slots, head_dim=128)[0].shape == (0, 2, 128)
    tables = torch.zeros((0, 3), dtype=torch.int32, device="cuda")
    lens = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert q4_cache.attention(none, kp, vp, tables, lens).shape == (0, 2, 128)
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    tables = torch.zeros((3, 0), dtype=torch.int32, device="cuda")
    out, lse = q4_cache.attention(randn((3, 2, 128), torch.bfloat16, 1), kp, vp, tables, lens,
                                  return_lse=True)
    assert not out.any() and torch.isinf(lse).all()


def test_refusals_on_device_tensors():
    kp, vp, tables, lengths, _ = make_cache([20, 20], 2, 128, 16, 140)
    q = randn((2, 4, 128), torch.bfloat16, 141)
    att = lambda **kw: q4_cache.attention(**{**dict(  # noqa: E731
        query=q, key_pages=kp, value_pages=vp, block_tables=tables, seq_lens=lengths), **kw})
    for bad in (dict(query=q[:, :3]), dict(query=q[0]), dict(block_tables=tables.long()),
                dict(seq_lens=lengths.long()), dict(seq_lens=lengths[:1]), dict(window=0),
                dict(sinks=-1), dict(scale=float("nan")), dict(query=q.transpose(1, 2)),
                dict(out=q.float()), dict(out=q[:1]), dict(query_starts=lengths),
                dict(block_tables=tables.cpu()), dict(query=q.cpu()),
                dict(query=torch.cat([q, q[:1]])), dict(key_pages=kp[..., :-1]), dict(out=q)):
        with pytest.raises(ValueError):
            att(**bad)
    for bad in (dict(query=q.float()), dict(key_pages=kp.view(torch.int8))):
        with pytest.raises(TypeError):
            att(**bad)
    rows, slots = randn((2, 2, 128), torch.bfloat16, 142), torch.arange(2, device="cuda")
    for bad in (dict(slots=slots.int()), dict(slots=slots[:1]), dict(slots=slots.cpu()),
                dict(value=rows[:1]), dict(key=rows.transpose(0, 2)), dict(value_pages=kp)):
        with pytest.raises(ValueError):
            q4_cache.write(**{**dict(key=rows, value=rows, key_pages=kp, value_pages=vp,
                                     slots=slots), **bad})
    with pytest.raises(TypeError):
        q4_cache.write(rows, rows.half(), kp, vp, slots)
    with pytest.raises(ValueError, match="overlap"):
        q4_cache.read(kp, vp, slots, head_dim=128, out=(rows, rows))
    with pytest.raises(RuntimeError, match="gradient"):
        q4_cache.write(rows.clone().requires_grad_(), rows, kp, vp, slots)
    with pytest.raises(TypeError):
        q4_cache.read(kp, vp, slots, head_dim=128, dtype=torch.float64)


def test_a_request_is_written_swapped_and_attended_to():
    """The operators together, as a server uses them: a prompt is written and
    attended to, its pages (all layers) go to host rows and come back to other
    blocks, and decoding goes on there with the same results."""
    layers, heads, kv_heads, dim, block, blocks = 3, 8, 2, 128, 16, 24
    n = 100
    need = -(-(n + 1) // block)
    caches = [q4_cache.allocate(blocks, block, kv_heads, dim) for _ in range(layers)]
    first = torch.randperm(blocks, generator=gen(150), device="cuda")[:need]
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")

    def slots_of(ids, count, at=0):
        j = torch.arange(at, at + count, device="cuda")
        return ids[j // block] * block + j % block

    for i, (kp, vp) in enumerate(caches):
        key, value = randn((n, kv_heads, dim), torch.bfloat16, 151 + i), \
            randn((n, kv_heads, dim), torch.bfloat16, 161 + i)
        q4_cache.write(key, value, kp, vp, slots_of(first, n))
        check(randn((n, heads, dim), torch.bfloat16, 171 + i), kp, vp, first[None].int(), lens, starts)
    tensors = [t for pair in caches for t in pair]
    page = tensors[0][0].numel()
    segments, composite = swapper.make_segments(
        [((f"t{i}",), t.numel()) for i, t in enumerate(tensors)], blocks)
    assert composite == 2 * layers * page
    pool = torch.zeros(need * composite, dtype=torch.uint8).pin_memory()
    sw = swapper.KVSwapper(0, segments, [t.view(-1) for t in tensors],
                           [frozenset({0})] * len(tensors), [1], kv_swap=pool)
    query = [randn((1, heads, dim), torch.bfloat16, 181 + i) for i in range(layers)]
    new = [(randn((1, kv_heads, dim), torch.bfloat16, 191 + i),
            randn((1, kv_heads, dim), torch.bfloat16, 201 + i)) for i in range(layers)]

    def turn(ids):
        got = []
        for i, (kp, vp) in enumerate(caches):
            q4_cache.write(*new[i], kp, vp, slots_of(ids, 1, n))
            got.append(q4_cache.attention(query[i], kp, vp, ids[None].int(), lens + 1))
        return got

    rows, zero, one = list(range(need)), [0] * need, [1] * need
    sw.swap_blocks([0], first.tolist(), rows, zero, zero, one, [None], False).synchronize()
    want = turn(first)
    for t in tensors:
        t.fill_(0xFF)
    second = torch.randperm(blocks, generator=gen(152), device="cuda")[:need]
    sw.swap_blocks([0], rows, second.tolist(), zero, zero, one, [None], True).synchronize()
    got = turn(second)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    sw.close()
    # the per-tensor swap op, which takes elements for 2 bytes
    kp = caches[0][0]
    host = torch.zeros((need, kp[0].numel() // 2), dtype=torch.int16).pin_memory()
    ops.swap(second.tolist(), rows, False, kp.view(blocks, -1).view(torch.int16), host)
    torch.cuda.synchronize()
    assert torch.equal(host.view(torch.uint8), kp[second].view(need, -1).cpu())
