"""GPU tests of the 4-bit cache where its numbers and its memory are easily got
wrong: rows at the ends of the value range, value scales far apart, weights and
queries of extreme size, and arguments that share memory.

Expected values come from the definition in 64 bits (q4_oracle)."""

import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

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


# ---- value scales far apart ---------------------------------------------------------


def attention_bound(query, kp, vp, tables, lens, starts=None, window=None, sinks=0):
    """(out, bound) from the definition, where every term of the bound carries its
    token's weight, so that what nobody attends to allows no error.

    With w the weights (sum 1), s and z the value scales and zeros:
      * a weight is off by dx, relatively: the score's (dim/16 + 4) 2^-23 max_j sum_d
        |q_d| (s c_d + |z|) scale (products summed in 32 bits in dim/16 steps, three
        more roundings, whole steps because an accumulation may truncate) and the
        hardware's exp2, 2^-21.  The normalised sum moves by at most
        2 dx sum_j w_j |v_j - out|;
      * each product w_j s_j is rounded once to fp16: 2^-11 of it, times the
        distance of a code from the middle, at most 8.  The largest product lies above 2^5
        before that rounding, so those below fp16's normal numbers are off by 2^-25 each, 2^-30
        of the largest; twice, since they may be scaled once more;
      * n/8 + 64 roundings of 2^-24 in sums of w_j (15 s_j + |z_j|), doubled for the part of
        the middle, which cancels;
      * the rounding to the output's type, and fp16's smallest half step.
    """
    tokens, heads, dim = query.shape
    group = heads // kp.shape[1]
    q = query.double().cpu()
    parts = [*q4_oracle.split(kp, dim), *q4_oracle.split(vp, dim)]
    block = parts[0].shape[2]
    lens, tables = lens.tolist(), tables.tolist()
    per = tokens // len(lens)
    starts = [i * per for i in range(len(lens) + 1)] if starts is None else starts.tolist()
    out = torch.zeros(tokens, heads, dim, dtype=torch.float64)
    bound = torch.zeros_like(out)
    half = torch.finfo(query.dtype).eps / 2
    for b, n in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        ids = tables[b][: -(-n // block)]
        kc, ks, kz, vc, vs, vz = (t[ids].transpose(0, 1).flatten(1, 2)[:, :n].double() for t in parts)
        p, j = torch.arange(n - (hi - lo), n)[:, None], torch.arange(n)[None]
        seen = j <= p
        if window:
            seen &= (j > p - window) | (j < sinks)
        for h in range(heads):
            kv = h // group
            x = q[lo:hi, h]
            k, v = kc[kv] * ks[kv][:, None] + kz[kv][:, None], vc[kv] * vs[kv][:, None] + vz[kv][:, None]
            score = (x @ k.T / math.sqrt(dim)).masked_fill(~seen, -math.inf)
            size = x.abs() @ (kc[kv] * ks[kv][:, None] + kz[kv].abs()[:, None]).T / math.sqrt(dim)
            dx = (dim / 16 + 4) * 2.0 ** -23 * size.masked_fill(~seen, 0).amax(1) + 2.0 ** -21
            w = torch.softmax(score, 1)
            o = w @ v
            spread = torch.stack([w[i] @ (v - o[i]).abs() for i in range(hi - lo)])
            step = w * vs[kv]
            e = 2 * dx[:, None] * spread
            e = e + (8 * 2.0 ** -11 * step.sum(1) + 8 * n * 2.0 ** -29 * step.amax(1))[:, None]
            e = e + (2 * (n / 8 + 64) * 2.0 ** -24 * (w @ (15 * vs[kv] + vz[kv].abs())))[:, None]
            out[lo:hi, h] = o
            bound[lo:hi, h] = e + half * (o.abs() + e) + (2.0 ** -25 if query.dtype is torch.float16 else 0)
    return out, bound


def steered_cache(lens, special, kv_heads, dim, block, small, seed):
    """A cache whose values have the scale `small` but for single tokens.  special:
    {(sequence, token): (push, rows)}: the key is -push in 16 channels where the queries are
    about 2, and `rows` is the token's value row."""
    need = [-(-n // block) for n in lens]
    shape = (sum(need) + 1, kv_heads, q4_cache.head_bytes(block, dim))
    kp, vp = (torch.full(shape, 0xFF, dtype=torch.uint8, device="cuda") for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(seed)
    order = torch.randperm(shape[0], generator=g, device="cuda")
    tables = torch.zeros((len(lens), max(need)), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(lens):
        ids = order[at:at + need[b]]
        at += need[b]
        tables[b, :need[b]] = ids.int()
        j = torch.arange(n, device="cuda")
        key = randn((n, kv_heads, dim), torch.float32, seed + 2 * b + 1)
        # a row's values step through the sixteen codes: scale `small`, exact
        value = (torch.randint(0, 16, (n, kv_heads, dim), generator=g, device="cuda") - 7.5) * small
        value[..., 0], value[..., 1] = -7.5 * small, 7.5 * small
        for (seq, token), (push, rows) in special.items():
            if seq == b:
                key[token] = 0
                key[token, :, :16] = -push
                value[token] = rows
        q4_cache.write(key, value, kp, vp, ids[j // block] * block + j % block)
    return kp, vp, tables, torch.tensor(lens, dtype=torch.int32, device="cuda")


def steered_queries(tokens, heads, dim, dtype, seed):
    q = randn((tokens, heads, dim), torch.float32, seed)
    q[..., :16] = 2 + 0.1 * q[..., :16]
    return q.to(dtype)


def hold(query, kp, vp, tables, lens, starts=None, **kw):
    got = q4_cache.attention(query, kp, vp, tables, lens, query_starts=starts, **kw).double().cpu()
    want, bound = attention_bound(query, kp, vp, tables, lens, starts, **kw)
    off = (got - want).abs()
    assert (off <= bound).all(), f"off by {(off / bound.clamp(min=1e-30)).max()} bounds"


def wide_row(scale, dim):
    """A value row with that scale: all codes appear."""
    return (torch.arange(dim, device="cuda") % 16 - 7.5) * scale


# Scales of the token that nobody attends to (weight about 1e-18) and of the others.
FAR_SCALES = [(0, -14), (4, -17), (10, -14), (13, -14), (13, -17)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("large,small", FAR_SCALES)
@pytest.mark.parametrize("heads,kv_heads,dim,block", [
    (4, 2, 64, 16), (7, 1, 128, 16), (12, 1, 128, 32), (32, 1, 128, 16), (4, 4, 256, 16), (12, 1, 256, 16)])
def test_decode_with_a_far_value_scale(dtype, large, small, heads, kv_heads, dim, block):
    """Wherever the token is: in the first unit, behind others, in the last one."""
    lens = [100, 200, 333]
    row = wide_row(2.0 ** large, dim)
    special = {(0, 0): (15.0, row), (1, 111): (15.0, row), (2, 331): (15.0, row)}
    cache = steered_cache(lens, special, kv_heads, dim, block, 2.0 ** small, 10)
    hold(steered_queries(len(lens), heads, dim, dtype, 20), *cache)


def test_far_value_scales_in_the_parts_of_a_long_sequence():
    """Pieces of one sequence, with and without such a token, that are joined."""
    row = wide_row(2.0 ** 13, 128)
    special = {(0, 5): (15.0, row), (0, 3000): (15.0, row), (0, 4998): (15.0, row)}
    cache = steered_cache([5000], special, 1, 128, 16, 2.0 ** -14, 30)
    for dtype in DTYPES:
        hold(steered_queries(1, 7, 128, dtype, 31), *cache)


@pytest.mark.parametrize("large,small", FAR_SCALES)
def test_a_scale_that_only_other_rows_see(large, small):
    """Several queries share a tile; the last token is seen by the last of them alone."""
    row = wide_row(2.0 ** large, 128)
    lens = [60, 160]
    cache = steered_cache(lens, {(0, 59): (15.0, row), (1, 157): (0.0, row)}, 2, 128, 16,
                          2.0 ** small, 40)
    hold(steered_queries(8, 6, 128, torch.float16, 41), *cache)
    hold(steered_queries(8, 6, 128, torch.bfloat16, 42), *cache, window=30, sinks=3)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("large,small", FAR_SCALES)
def test_many_rows_with_a_far_value_scale(large, small, dim):
    """The kernel of many rows: rows that see the token and rows that do not."""
    heads, kv_heads, lens, counts = 32, 16, [340, 300], [340, 150]
    assert sum(counts) * (heads // kv_heads) // 128 * kv_heads >= 74
    row = wide_row(2.0 ** large, dim)
    special = {(0, 0): (15.0, row), (0, 200): (15.0, row), (1, 140): (15.0, row),
               (1, 299): (0.0, row)}
    cache = steered_cache(lens, special, kv_heads, dim, 16, 2.0 ** small, 50)
    starts = torch.tensor([0, 340, 490], dtype=torch.int32, device="cuda")
    hold(steered_queries(490, heads, dim, torch.float16, 51), *cache, starts=starts)
    hold(steered_queries(490, heads, dim, torch.bfloat16, 52), *cache, starts=starts, window=90, sinks=2)


@pytest.mark.parametrize("push", [-5.0, 0.0])
def test_a_token_without_values_that_takes_the_weight(push):
    """A row of zeros with nearly all of the weight (push -5: 1 - 2^-16 of it): what is left
    of the other tokens is the whole output."""
    zero = torch.zeros(128, device="cuda")
    cache = steered_cache([150, 40], {(0, 0): (push, zero), (1, 20): (push, zero)}, 1, 128, 16, 1.0, 60)
    hold(steered_queries(2, 7, 128, torch.bfloat16, 61), *cache)
    cache = steered_cache([320], {(0, 0): (push, zero)}, 16, 128, 16, 1.0, 62)
    hold(steered_queries(320, 32, 128, torch.bfloat16, 63), *cache)


def test_log_sum_exp_with_any_value_scale():
    """The log-sum-exp does not depend on the values.  Bound: the score's error, and
    one rounding of the result's size, in a logarithm that is off by 2^-22."""
    query = steered_queries(2, 7, 128, torch.float16, 71)
    many = steered_queries(320, 32, 128, torch.float16, 73)
    for small in (0.0, 2.0 ** -17, 1.0, 2.0 ** 12):
        for q, lens, kv_heads in ((query, [150, 2000], 1), (many, [320], 16)):
            cache = steered_cache(lens, {}, kv_heads, 128, 16, small, 70)
            _, lse = q4_cache.attention(q, *cache, return_lse=True)
            _, want, _, bound = q4_oracle.attention(q, *cache)
            assert ((lse.double().cpu() - want).abs() <= bound).all()


# ---- rows marked as NaN ---------------------------------------------------------------


@pytest.mark.parametrize("push", [0.0, 60.0])
@pytest.mark.parametrize("token", [3, 70, 145, 2500])
def test_a_nan_value_reaches_every_row_that_sees_it(token, push):
    """Even where the weight underflows (push 60: a weight of 2^-245): its product with a
    NaN is none the less a NaN, in masked tiles, in plain ones and in joined pieces."""
    bad = torch.full((128,), math.nan, device="cuda")
    n = 150 if token < 150 else 4000
    cache = steered_cache([n, 30], {(0, token): (push, bad)}, 1, 128, 16, 1.0, 80)
    q = steered_queries(8, 7, 128, torch.bfloat16, 81)  # positions n - 4 ... n - 1
    got = q4_cache.attention(q, *cache)
    sees = torch.arange(n - 4, n) >= token
    assert torch.equal(got[:4].isnan().all(-1).all(-1).cpu(), sees)
    assert torch.equal(got[:4].isnan().any(-1).any(-1).cpu(), sees)
    assert torch.isfinite(got[4:]).all()


@pytest.mark.parametrize("push", [0.0, 60.0])
def test_a_nan_value_among_many_rows(push):
    bad = torch.full((128,), math.nan, device="cuda")
    for token in (0, 131, 300):
        cache = steered_cache([340], {(0, token): (push, bad)}, 16, 128, 16, 1.0, 90)
        got = q4_cache.attention(steered_queries(340, 32, 128, torch.float16, 91), *cache)
        assert torch.isfinite(got[:token]).all()
        assert got[token:].isnan().all()
        got = q4_cache.attention(steered_queries(340, 32, 128, torch.float16, 92), *cache, window=40)
        assert got[token:token + 40].isnan().all()
        assert torch.isfinite(got[:token]).all() and torch.isfinite(got[token + 40:]).all()


def test_a_nan_value_in_a_stretch_without_weight():
    """Whole pieces of a long sequence whose weights underflow against the others'."""
    zero, bad = torch.zeros(128, device="cuda"), torch.full((128,), math.nan, device="cuda")
    stretch = {(0, t): (60.0, zero) for t in range(900, 1500)}
    q = steered_queries(1, 7, 128, torch.bfloat16, 95)
    hold(q, *steered_cache([4000], stretch, 1, 128, 16, 1.0, 96))
    stretch[0, 1200] = (60.0, bad)
    assert q4_cache.attention(q, *steered_cache([4000], stretch, 1, 128, 16, 1.0, 96)).isnan().all()


# ---- queries of any size --------------------------------------------------------------


@pytest.mark.parametrize("size,scale", [(5e37, 2e-38), (1e36, 1e-36), (1e-38, 1e37), (1e-37, 2e36)])
def test_queries_at_the_ends_of_bf16(size, scale):
    """With a softmax scale that brings the scores back, the definition is finite."""
    for q, lens, kv_heads in ((randn((2, 7, 128), torch.float32, 101), [150, 700], 1),
                              (randn((8, 4, 256), torch.float32, 102), [50, 90], 2),
                              (randn((340, 32, 128), torch.float32, 103), [340], 16)):
        q = (q.clamp(-5, 5) * size).to(torch.bfloat16)
        cache = steered_cache(lens, {}, kv_heads, q.shape[2], 16, 0.25, 100)
        got, lse = q4_cache.attention(q, *cache, scale=scale, return_lse=True)
        out, want, out_bound, lse_bound = q4_oracle.attention(q, *cache, scale=scale)
        assert ((got.double().cpu() - out).abs() <= out_bound).all()
        assert ((lse.double().cpu() - want).abs() <= lse_bound).all()


@pytest.mark.parametrize("size,small", [
    (3e5, 1.0), (1e6, 2.0 ** -17), (1e7, 1.0), (1e8, 2.0 ** -17), (1e9, 2.0 ** 12), (1e37, 1.0),
    (1e37, 2.0 ** -14)])
def test_scores_as_large_as_fp32_holds(size, small):
    """Where fp32 counts scores in whole numbers and more, the largest takes all.  Keys of
    codes 0 and 15 alone."""
    n, dim = 320, 128
    for tokens, heads, kv_heads in ((1, 7, 1), (320, 32, 16)):
        kp, vp, tables, lens = steered_cache([n], {}, kv_heads, dim, 16, small, 110)
        g = torch.Generator(device="cuda").manual_seed(112)
        key = torch.randint(0, 2, (n, kv_heads, dim), generator=g, device="cuda").float()
        key[..., 0], key[..., 1] = 0.0, 1.0
        j = torch.arange(n, device="cuda")
        slots = tables[0].long()[j // 16] * 16 + j % 16
        _, value = q4_cache.read(kp, vp, slots, head_dim=dim, dtype=torch.float32)
        q4_cache.write(key, value, kp, vp, slots)
        q = (randn((tokens, heads, dim), torch.float32, 111).clamp(-3, 3) * size).to(torch.bfloat16)
        got, lse = q4_cache.attention(q, kp, vp, tables, lens, return_lse=True)
        key, value = (t.double().repeat_interleave(heads // kv_heads, 1) for t in
                      q4_cache.read(kp, vp, slots, head_dim=dim, dtype=torch.float32))
        score = torch.einsum("thd,jhd->thj", q.double(), key) / math.sqrt(dim)
        place = torch.arange(n - tokens, n, device="cuda")
        score.masked_fill_((torch.arange(n, device="cuda") > place[:, None])[:, None], -math.inf)
        two = score.topk(2, -1).values
        # by how much a score is off: (dim/16 + 4) 2^-23 of the sum of |q| |k|
        off = torch.einsum("thd,jhd->thj", q.double().abs(), key.abs()).amax(-1) / math.sqrt(dim)
        off *= (dim / 16 + 4) * 2.0 ** -23
        clear = two[..., 0] - two[..., 1] > 4 * off + 40  # others weigh e^-40 at most
        assert clear[1 if tokens > 1 else 0:].double().mean() > 0.8
        want = value[score.argmax(-1), torch.arange(heads, device="cuda")]
        # half a step of bf16; fp16's half step 2^-25 in the weight of a code, 8 from the middle
        bound = 2.0 ** -8 * want.abs() + 8 * 2.0 ** -25 + 8 * 2.0 ** -11 * small
        assert torch.isfinite(got).all()
        assert ((got.double() - want).abs() <= bound)[clear].all()
        assert ((lse.double() - two[..., 0]).abs() <= off + 6 + 2.0 ** -22 * two[..., 0].abs()).all()


# ---- arguments that share memory -------------------------------------------------------


def test_outputs_that_share_memory_with_inputs_are_refused():
    block, dim = 16, 128
    kp, vp, tables, lens = steered_cache([40, 20], {}, 2, dim, block, 1.0, 120)
    qkv = randn((2, 8, dim), torch.bfloat16, 121)
    att = lambda q, out: q4_cache.attention(q, kp, vp, tables, lens, out=out)  # noqa: E731
    want = q4_cache.attention(qkv[:, :4].clone(), kp, vp, tables, lens)
    before = qkv.clone()
    for out in (qkv[:, :4], qkv[:, 1:5], qkv[:, 3:7]):
        with pytest.raises(ValueError, match="overlap"):
            att(qkv[:, :4], out)
    with pytest.raises(ValueError, match="overlap"):  # every row in one place
        att(qkv[:, :4], torch.empty((1, 4, dim), dtype=torch.bfloat16, device="cuda").expand(2, 4, dim))
    with pytest.raises(ValueError, match="overlap"):  # in the pages
        att(qkv[:, :4], kp.view(-1)[:2 * 4 * dim * 2].view(torch.bfloat16).view(2, 4, dim))
    numbers = torch.zeros(2 * 4 * dim, dtype=torch.int32, device="cuda")
    numbers[:2] = lens
    with pytest.raises(ValueError, match="overlap"):  # in the lengths
        q4_cache.attention(qkv[:, :4], kp, vp, tables, numbers[:2],
                           out=numbers.view(torch.bfloat16)[:2 * 4 * dim].view(2, 4, dim))
    assert torch.equal(qkv, before)
    assert torch.equal(att(qkv[:, :4], qkv[:, 4:]), want)  # beside the queries: allowed
    assert torch.equal(qkv[:, :4], before[:, :4]) and torch.equal(qkv[:, 4:], want)

    slots = torch.arange(3, device="cuda")
    rows = torch.zeros((3, 5, dim), dtype=torch.bfloat16, device="cuda")
    read = lambda a, b: q4_cache.read(kp, vp, slots, head_dim=dim, out=(a, b))  # noqa: E731
    for a, b in ((rows[:, :2], rows[:, 1:3]), (rows[:, 2:4], rows[:, 2:4]),
                 (rows[:1, :2].expand(3, 2, dim), rows[:, 2:4]),
                 (rows[:, :2], vp.view(-1)[:3 * 2 * dim * 2].view(torch.bfloat16).view(3, 2, dim))):
        with pytest.raises(ValueError, match="overlap"):
            read(a, b)
    plain = q4_cache.read(kp, vp, slots, head_dim=dim)
    got = read(rows[:, :2], rows[:, 2:4])
    assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1]) and not rows[:, 4].any()

    before = kp.clone()
    with pytest.raises(ValueError, match="overlap"):
        q4_cache.write(rows[:, :2], rows[:, 2:4], kp, kp[:], slots)
    inside = kp.view(-1)[:3 * 2 * dim * 2].view(torch.bfloat16).view(3, 2, dim)
    with pytest.raises(ValueError, match="overlap"):  # rows in the pages that are written
        q4_cache.write(inside, rows[:, :2], kp, vp, slots)
    with pytest.raises(ValueError, match="overlap"):
        q4_cache.write(rows[:, :2], rows[:, 2:4], kp, vp, kp.view(-1)[:24].view(torch.int64))
    assert torch.equal(kp, before)


def test_interleaved_caches_are_written_and_read():
    """Layers, keys and values side by side in one buffer, blocks outermost."""
    blocks, layers, block, heads, dim = 7, 3, 16, 2, 64
    buffer = torch.zeros((blocks, layers, 2, heads, q4_cache.head_bytes(block, dim)),
                         dtype=torch.uint8, device="cuda")
    slots = torch.randperm(blocks * block, device="cuda")[:50]
    for i in range(layers):
        key, value = randn((50, heads, dim), torch.float16, 130 + i), randn((50, heads, dim), torch.float16, 140 + i)
        q4_cache.write(key, value, buffer[:, i, 0], buffer[:, i, 1], slots)
        alone = q4_cache.allocate(blocks, block, heads, dim)
        q4_cache.write(key, value, *alone, slots)
        assert torch.equal(alone[0], buffer[:, i, 0]) and torch.equal(alone[1], buffer[:, i, 1])


# ---- what autograd has to know ----------------------------------------------------------


def test_forward_mode_gradients_are_refused():
    kp, vp, tables, lens = steered_cache([20, 20], {}, 2, 128, 16, 1.0, 155)
    slots = torch.arange(2, device="cuda")
    rows = randn((2, 2, 128), torch.bfloat16, 156)
    want = q4_cache.attention(rows, kp, vp, tables, lens)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(rows.clone(), rows)
        for call in (lambda: q4_cache.attention(dual, kp, vp, tables, lens),
                     lambda: q4_cache.attention(rows, kp, vp, tables, lens, out=dual),
                     lambda: q4_cache.read(kp, vp, slots, head_dim=128, out=(dual, rows.clone())),
                     lambda: q4_cache.write(rows, dual, kp, vp, slots)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        plain = forward_ad.unpack_dual(dual).primal
        assert torch.equal(q4_cache.attention(plain, kp, vp, tables, lens), want)



def test_autograd_sees_what_was_overwritten():
    """A tensor that a gradient needs and that an operator then writes to is noticed."""
    kp, vp, tables, lens = steered_cache([20, 20], {}, 2, 128, 16, 1.0, 150)
    slots = torch.arange(2, device="cuda")
    rows = randn((2, 2, 128), torch.bfloat16, 151)
    versions = kp._version, vp._version
    q4_cache.write(rows, rows, kp, vp, slots)
    assert kp._version > versions[0] and vp._version > versions[1]
    versions = kp._version, vp._version, rows._version
    q4_cache.read(kp, vp, slots, head_dim=128)
    q4_cache.attention(randn((2, 2, 128), torch.bfloat16, 152), kp, vp, tables, lens)
    assert (kp._version, vp._version, rows._version) == versions
    weight = torch.ones((2, 2, 128), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    query = randn((2, 2, 128), torch.bfloat16, 153)
    for overwrite in (lambda t: q4_cache.attention(query, kp, vp, tables, lens, out=t),
                      lambda t: q4_cache.read(kp, vp, slots, head_dim=128, out=(t, torch.empty_like(t))),
                      lambda t: q4_cache.read(kp, vp, slots, head_dim=128, out=(torch.empty_like(t), t))):
        saved = rows.clone()
        loss = (saved * weight).sum()
        overwrite(saved)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_inference_tensors():
    """Pages made in inference mode are used outside it, and the other way round."""
    slots = torch.arange(3, device="cuda")
    rows = randn((3, 2, 128), torch.bfloat16, 160)
    with torch.inference_mode():
        kp, vp = q4_cache.allocate(2, 16, 2, 128)
        q4_cache.write(rows, rows, kp, vp, slots)
    q4_cache.write(rows, rows, kp, vp, slots)
    a = q4_cache.read(kp, vp, slots, head_dim=128)
    kp, vp = q4_cache.allocate(2, 16, 2, 128)
    with torch.inference_mode():
        q4_cache.write(rows, rows, kp, vp, slots)
        b = q4_cache.read(kp, vp, slots, head_dim=128, out=(rows.clone(), rows.clone()))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ---- short caches in the kernel of many rows --------------------------------------------


@pytest.mark.parametrize("n", [1, 16, 100, 128, 129, 256, 257, 384, 385])
@pytest.mark.parametrize("queries", [64, 100])
def test_many_rows_over_few_blocks(n, queries):
    """One, two, three and four blocks of 128 tokens, for CTAs of one tile (64 queries of two
    heads) and of two.  Calls follow one another at once: nothing of a block that has ended
    may reach the next one."""
    cache = steered_cache([n], {}, 148, 64, 16, 0.5, 170)
    q = steered_queries(queries, 296, 64, torch.float16, 171)
    results = [q4_cache.attention(q, *cache) for _ in range(6)]
    for r in results[1:]:
        assert torch.equal(r, results[0])
    some = slice(0, 4)  # two kv heads hold for all
    pages = [p[:, :2].contiguous() for p in cache[:2]]
    want, _, bound, _ = q4_oracle.attention(q[:, some], *pages, *cache[2:])
    assert ((results[0][:, some].double().cpu() - want).abs() <= bound).all()


# ---- lengths, starts and values that the documentation speaks of -------------------------


def test_values_beyond_fp16_when_read():
    """Scale and zero are rounded, so a row's highest value may lie above 65504: fp16 has
    no number for those from 65520 on and gives infinity, bfloat16 and float32 keep them."""
    x = torch.linspace(-1, 1, 128, device="cuda")[None, None] * 65504
    kp, vp = q4_cache.allocate(1, 16, 1, 128)
    slots = torch.zeros(1, dtype=torch.int64, device="cuda")
    q4_cache.write(x, x, kp, vp, slots)
    exact = q4_oracle.values(kp, 128)[0, 0, 0]
    assert exact.max() == 65536.0
    for dtype in DTYPES + [torch.float32]:
        key, _ = q4_cache.read(kp, vp, slots, head_dim=128, dtype=dtype)
        assert torch.equal(key[0, 0].cpu(), exact.to(dtype))
        assert torch.isfinite(key).all() == (dtype is not torch.float16)


def test_lengths_and_starts_outside_their_range():
    """A length above the table's is cut and reported; one below zero counts as zero and
    starts outside the query are cut, both without a report."""
    kp, vp, tables, lens = steered_cache([48, 20], {}, 2, 128, 16, 1.0, 180)
    q = steered_queries(4, 4, 128, torch.bfloat16, 181)
    want = q4_cache.attention(q, kp, vp, tables, lens)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = q4_cache.attention(q, kp, vp, tables, ints(48, -2 ** 31))
    assert torch.equal(got[:2], want[:2]) and not got[2:].any()
    inside = q4_cache.attention(q, kp, vp, tables, lens, query_starts=ints(0, 2, 4))
    got = q4_cache.attention(q, kp, vp, tables, lens, query_starts=ints(-5, 2, 2 ** 31 - 1))
    assert torch.equal(got, inside)
    assert _lib.device_status(0) == 0
    tables[1] = tables[0]
    got = q4_cache.attention(q, kp, vp, tables, ints(48, 2 ** 31 - 1))
    assert _lib.device_status(0, reset=True) == _lib.KVX_ERR_EXTENT
    assert torch.equal(got, q4_cache.attention(q, kp, vp, tables, ints(48, 48)))


# ---- rows keep to themselves ---------------------------------------------------------------


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_query_that_is_no_number_spoils_its_row_alone(bad):
    for tokens, heads, kv_heads, lens in ((8, 7, 1, [150, 700]), (340, 32, 16, [340])):
        cache = steered_cache(lens, {}, kv_heads, 128, 16, 1.0, 190)
        q = steered_queries(tokens, heads, 128, torch.bfloat16, 191)
        want, want_lse = q4_cache.attention(q, *cache, return_lse=True)
        q[1, 2, 77] = bad
        got, lse = q4_cache.attention(q, *cache, return_lse=True)
        assert got[1, 2].isnan().all() and lse[1, 2].isnan()
        got[1, 2], lse[1, 2] = want[1, 2], want_lse[1, 2]
        # Another row's reference point may move earlier or later: a rounding, not the row's number.
        assert torch.allclose(got.float(), want.float(), rtol=2.0 ** -7, atol=2.0 ** -9)
        assert torch.allclose(lse, want_lse, rtol=0, atol=2.0 ** -18)


def test_rows_of_any_size_in_one_tile():
    """Rows whose scores are far beyond fp32's fractions beside ordinary ones, in one call,
    and a scale of either sign."""
    for tokens, heads, kv_heads, lens in ((8, 7, 1, [150, 700]), (340, 32, 16, [340])):
        cache = steered_cache(lens, {}, kv_heads, 128, 16, 1.0, 195)
        q = steered_queries(tokens, heads, 128, torch.bfloat16, 196)
        for scale in (None, -0.05):
            want, want_lse = q4_cache.attention(q, *cache, scale=scale, return_lse=True)
            mixed = q.clone()
            mixed[0::2, 0::3] *= 1e9
            got, lse = q4_cache.attention(mixed, *cache, scale=scale, return_lse=True)
            same = torch.ones(q.shape[:2], dtype=torch.bool, device="cuda")
            same[0::2, 0::3] = False
            assert torch.isfinite(got).all() and torch.isfinite(lse).all()
            assert torch.allclose(got[same].float(), want[same].float(), rtol=2.0 ** -7, atol=2.0 ** -9)
            assert torch.allclose(lse[same], want_lse[same], rtol=0, atol=2.0 ** -18)


def test_a_scale_of_zero_is_the_mean():
    for tokens, heads, kv_heads, lens in ((2, 7, 1, [150, 700]), (340, 32, 16, [340])):
        cache = steered_cache(lens, {}, kv_heads, 128, 16, 1.0, 197)
        q = steered_queries(tokens, heads, 128, torch.bfloat16, 198)
        got, lse = q4_cache.attention(q, *cache, scale=0.0, return_lse=True)
        want, want_lse, bound, lse_bound = q4_oracle.attention(q, *cache, scale=0.0)
        assert ((got.double().cpu() - want).abs() <= bound).all()
        assert ((lse.double().cpu() - want_lse).abs() <= lse_bound).all()
