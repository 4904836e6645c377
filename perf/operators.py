"""The operators of the 4-bit paged KV cache, as a serving program calls them.

A cache page holds one block of one tensor (K or V) in 4 bits: for each kv head the codes of the block's
tokens (two to a byte, the even dimension in the low nibble), then for each token an fp16 scale and an fp16
zero.  Three operators work on it: ``write`` quantises new rows into their slots, ``read`` gives rows back,
``attention`` attends over the cache through block tables.

``own`` false: elementary torch operations in 32 bits (64 where a code is chosen).  ``own`` true: the
framework's entry points in ``aegaeon_b200.q4_cache``.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LIMIT = 65504.0  # largest finite fp16: scale and zero are held in that type


def listed():
    return [
        # A prompt's rows as they leave a fused QKV projection (28 query heads, 4 kv heads), odd length,
        # a few padded rows that belong to no slot.
        dict(name="write_fused_odd", kind="write", tokens=1037, kv_heads=4, head_dim=128, block=16, dtype="bf16",
             fused=28, padded=13),
        # A batch of prompts of a 32-head model written in one call.
        dict(name="write_prompts", kind="write", tokens=8192, kv_heads=32, head_dim=128, block=16, dtype="fp16",
             fused=0, padded=0),
        # One request read back into 16 bits, small heads, larger blocks.
        dict(name="read_request", kind="read", tokens=777, kv_heads=8, head_dim=64, block=32, dtype="fp16"),
        # A batch of requests read back (a 16-bit engine takes them over).
        dict(name="read_requests", kind="read", tokens=65536, kv_heads=8, head_dim=128, block=16, dtype="bf16"),
        # One decode turn of a single short request: its new row is written, then read by the attention.
        # Latency counts.
        dict(name="turn_one", kind="turn", batch=1, length=1025, spread=0.0, queries=1, heads=28, kv_heads=4,
             head_dim=128, block=16, dtype="bf16", window=0, sinks=0, padded=0, lse=False),
        # One decode turn of a ragged batch, padded to the size that a captured graph has.
        dict(name="turn_batch", kind="turn", batch=32, length=4096, spread=0.95, queries=1, heads=32, kv_heads=8,
             head_dim=128, block=16, dtype="bf16", window=0, sinks=0, padded=3, lse=False),
        # Decode of a model without grouped heads.
        dict(name="decode_ungrouped", kind="attention", batch=16, length=2048, spread=0.5, queries=1, heads=32,
             kv_heads=32, head_dim=128, block=16, dtype="fp16", window=0, sinks=0, padded=0, lse=False),
        # Decode of one very long request: the work has to be split along the cache.
        dict(name="decode_long", kind="attention", batch=1, length=131072, spread=0.0, queries=1, heads=28,
             kv_heads=4, head_dim=128, block=16, dtype="bf16", window=0, sinks=0, padded=0, lse=True),
        # Decode of a large batch of long requests: the largest read of a cache.
        dict(name="decode_large", kind="attention", batch=128, length=8192, spread=0.5, queries=1, heads=32,
             kv_heads=8, head_dim=128, block=16, dtype="bf16", window=0, sinks=0, padded=0, lse=False),
        # Four tokens a request checked at once (speculative decoding), sliding window with four sinks.
        dict(name="verify_window", kind="attention", batch=24, length=20000, spread=0.9, queries=4, heads=32,
             kv_heads=8, head_dim=64, block=32, dtype="fp16", window=4096, sinks=4, padded=0, lse=True),
        # Pieces of prompts of odd lengths behind a cached prefix, sliding window with sinks.
        dict(name="extend_window", kind="extend", batch=3, length=5003, spread=0.6, queries=411, heads=28,
             kv_heads=4, head_dim=128, block=16, dtype="bf16", window=1024, sinks=4, padded=1, lse=True),
        # Long pieces of prompts behind long cached prefixes: bound by the products.
        dict(name="extend_large", kind="extend", batch=4, length=8192, spread=0.0, queries=1024, heads=32,
             kv_heads=8, head_dim=128, block=16, dtype="bf16", window=0, sinks=0, padded=0, lse=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["write", "read", "turn", "attention", "attention", "extend"])
    dtype = rng.choice(["bf16", "fp16"])
    head_dim = rng.choice([64, 128, 128])
    block = rng.choice([16, 16, 32, 64, 128])
    if kind in ("write", "read"):
        kv_heads = rng.choice([1, 2, 4, 8, 16, 32])
        tokens = _log(rng, 1, min(65536, 2 ** 25 // (kv_heads * head_dim)))
        case = dict(kind=kind, tokens=tokens, kv_heads=kv_heads, head_dim=head_dim, block=block,
                    dtype=rng.choice([dtype, dtype, "fp32"]) if kind == "write" else dtype)
        if kind == "write":
            case.update(fused=rng.choice([0, kv_heads, 4 * kv_heads]), padded=rng.choice([0, 0, tokens // 9]))
        return case
    kv_heads, group = rng.choice([(1, 8), (2, 6), (4, 7), (8, 4), (8, 4), (8, 8), (16, 1), (16, 2), (32, 1)])
    lse = rng.random() < 0.4
    window = rng.choice([0, 0, _log(rng, 16, 4096)])
    sinks = rng.choice([0, 1, 4, 37]) if window else 0
    case = dict(kind=kind, head_dim=head_dim, block=block, dtype=dtype, heads=kv_heads * group, kv_heads=kv_heads,
                window=window, sinks=sinks, lse=lse, spread=rng.choice([0.0, round(rng.random(), 2)]),
                padded=rng.choice([0, 0, 1]))
    if kind == "extend":
        batch = rng.choice([1, 2, 3, 5])
        length = _log(rng, 48, 8192)
        most = 2 ** 30 // (case["heads"] * length * batch)
        case.update(batch=batch, length=length, queries=min(length, _log(rng, 17, max(18, min(2048, most)))))
    else:
        batch = _log(rng, 1, 128)
        length = _log(rng, 1, min(131072, 2 ** 29 // (batch * kv_heads * head_dim)))
        case.update(batch=batch, length=length, queries=1 if kind == "turn" else rng.choice([1, 1, 2, 4]))
    return case


# ---- inputs -----------------------------------------------------------------------------------------------


def _spread(i, spread):
    return 1.0 - spread * (0.6180339887498949 * i % 1.0)


def _lengths(case):
    """Tokens in the cache of each sequence, this call's own among them; padded ones have none."""
    got = [max(1, int(round(case["length"] * _spread(i, case["spread"])))) for i in range(case["batch"])]
    return got[: case["batch"] - case["padded"]] + [0] * min(case["padded"], case["batch"])


def _queries(case):
    """Query tokens of each sequence."""
    if case["kind"] != "extend":
        return [case["queries"]] * case["batch"]
    return [min(n, max(1, int(round(case["queries"] * _spread(3 * i + 1, case["spread"]))))) if n else 0
            for i, n in enumerate(_lengths(case))]


def _normal(shape, g, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _rows(tokens, case, g, key):
    """K or V rows as projections give them: a few strong channels in K, an offset by channel in V."""
    shape = (tokens, case["kv_heads"], case["head_dim"])
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    channel = torch.randn(shape[1:], generator=g, device="cuda", dtype=torch.float32)
    x = x * (1 + 2 * (channel > 1.8)) if key else x + 0.3 * channel
    return x.to(torch.float16 if case["dtype"] == "fp16" else torch.bfloat16)


def _pool(blocks, case, g, key):
    """Pages of a cache in use."""
    block, dim = case["block"], case["head_dim"]
    pages = torch.empty((blocks, case["kv_heads"], block * (dim // 2 + 4)), device="cuda", dtype=torch.uint8)
    step = max(1, 2 ** 25 // (block * case["kv_heads"] * dim))
    for at in range(0, blocks, step):
        n = min(step, blocks - at)
        _store(pages, _rows(n * block, case, g, key),
               torch.arange(at * block, (at + n) * block, device="cuda"), block)
    return pages


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    block, dim, kv_heads = case["block"], case["head_dim"], case["kv_heads"]
    s = dict(kind=case["kind"], block=block, head_dim=dim, dtype=DTYPES[case["dtype"]])
    if case["kind"] in ("write", "read"):
        tokens = case["tokens"]
        need = -(-tokens // block)
        blocks = need + need // 8 + 1
        order = torch.randperm(blocks, generator=g, device="cuda")[:need]
        slots = (order[:, None] * block + torch.arange(block, device="cuda")).reshape(-1)[:tokens]
        s["slots"] = slots.contiguous()
        if case["kind"] == "read":
            s["key_pages"], s["value_pages"] = _pool(blocks, case, g, True), _pool(blocks, case, g, False)
            return s
        shape = (blocks, kv_heads, block * (dim // 2 + 4))
        s["key_pages"] = torch.zeros(shape, device="cuda", dtype=torch.uint8)
        s["value_pages"] = torch.zeros(shape, device="cuda", dtype=torch.uint8)
        if case["fused"]:
            q = _normal((tokens, case["fused"], dim), g, s["dtype"])
            qkv = torch.cat([q, _rows(tokens, case, g, True).to(s["dtype"]), _rows(tokens, case, g, False).to(s["dtype"])], 1)
            s["key"], s["value"] = qkv[:, case["fused"]:case["fused"] + kv_heads], qkv[:, case["fused"] + kv_heads:]
        else:
            s["key"], s["value"] = _rows(tokens, case, g, True).to(s["dtype"]), _rows(tokens, case, g, False).to(s["dtype"])
        if case["padded"]:
            s["slots"][-case["padded"]:] = -1
        return s
    lengths, queries = _lengths(case), _queries(case)
    need = [-(-n // block) for n in lengths]
    width, blocks = max(1, max(need)), sum(need) + sum(need) // 8 + 1
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    tables = torch.zeros((case["batch"], width), device="cuda", dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = order[at:at + n]
        at += n
    s["key_pages"], s["value_pages"] = _pool(blocks, case, g, True), _pool(blocks, case, g, False)
    s["tables"], s["lengths"] = tables, torch.tensor(lengths, device="cuda", dtype=torch.int32)
    s["window"], s["sinks"], s["lse"] = case["window"] or None, case["sinks"], case["lse"]
    s["query"] = _normal((sum(queries), case["heads"], dim), g, s["dtype"])
    s["starts"] = None
    if case["kind"] == "extend":
        starts = [0]
        for n in queries:
            starts.append(starts[-1] + n)
        s["starts"] = torch.tensor(starts, device="cuda", dtype=torch.int32)
        s["most"] = max(queries)
    else:
        s["most"] = case["queries"]
    if case["kind"] == "turn":
        s["key"], s["value"] = _rows(case["batch"], case, g, True), _rows(case["batch"], case, g, False)
        last = (s["lengths"].long() - 1).clamp(min=0)
        slots = tables.gather(1, (last // block)[:, None])[:, 0].long() * block + last % block
        s["slots"] = torch.where(s["lengths"] > 0, slots, torch.full_like(slots, -1))
    return s


# ---- one pass ---------------------------------------------------------------------------------------------


def run(s):
    if own:
        return _run_own(s)
    if s["kind"] in ("write", "turn"):
        _store(s["key_pages"], s["key"], s["slots"], s["block"])
        _store(s["value_pages"], s["value"], s["slots"], s["block"])
    if s["kind"] in ("write", "read"):
        return {"key": _load(s["key_pages"], s["slots"], s["block"], s["head_dim"]).to(s["dtype"]),
                "value": _load(s["value_pages"], s["slots"], s["block"], s["head_dim"]).to(s["dtype"])}
    out, lse = _attend(s)
    got = {"out": out, "lse": lse} if s["lse"] else {"out": out}
    if s["kind"] == "turn":  # the rows as the cache now holds them
        got.update(key=_load(s["key_pages"], s["slots"], s["block"], s["head_dim"]).to(s["dtype"]),
                   value=_load(s["value_pages"], s["slots"], s["block"], s["head_dim"]).to(s["dtype"]))
    return got


def _run_own(s):
    from aegaeon_b200 import q4_cache

    if s["kind"] in ("write", "turn"):
        q4_cache.write(s["key"], s["value"], s["key_pages"], s["value_pages"], s["slots"])
    if s["kind"] in ("write", "read"):
        key, value = q4_cache.read(s["key_pages"], s["value_pages"], s["slots"], head_dim=s["head_dim"],
                                   dtype=s["dtype"])
        return {"key": key, "value": value}
    got = q4_cache.attention(s["query"], s["key_pages"], s["value_pages"], s["tables"], s["lengths"],
                             query_starts=s["starts"], window=s["window"], sinks=s["sinks"], return_lse=s["lse"])
    got = {"out": got[0], "lse": got[1]} if s["lse"] else {"out": got}
    if s["kind"] == "turn":
        got["key"], got["value"] = q4_cache.read(s["key_pages"], s["value_pages"], s["slots"],
                                                 head_dim=s["head_dim"], dtype=s["dtype"])
    return got


# ---- the plain forms --------------------------------------------------------------------------------------


def _parts(pages, block, dim):
    """Views of pages [..., bytes]: codes [..., block, dim / 2] and (scale, zero) [..., block, 2]."""
    codes = pages[..., : block * dim // 2].unflatten(-1, (block, dim // 2))
    params = pages[..., block * dim // 2:].view(torch.float16).unflatten(-1, (block, 2))
    return codes, params


def _store(pages, rows, slots, block):
    """Quantises rows [tokens, kv_heads, dim] into their slots; negative slots are skipped."""
    dim = rows.shape[-1]
    keep = slots >= 0
    rows, slots = rows[keep].float(), slots[keep]
    finite = torch.isfinite(rows).all(-1, keepdim=True)
    rows = rows.clamp(-LIMIT, LIMIT)
    low, high = rows.amin(-1, keepdim=True), rows.amax(-1, keepdim=True)
    scale = ((high - low) / 15).half()
    zero = low.half()
    # In 64 bits: which side of a border between two codes a value is on.
    code = torch.round((rows.double() - zero.double()) / scale.double()).clamp(0, 15)
    code = torch.where(finite & (scale > 0), code, torch.zeros_like(code)).to(torch.uint8)
    params = torch.where(finite, torch.cat([scale, zero], -1), torch.full_like(zero, math.nan))
    to_codes, to_params = _parts(pages, block, dim)
    at, within = slots // block, slots % block
    to_codes[at, :, within] = code[..., 0::2] | (code[..., 1::2] << 4)
    to_params[at, :, within] = params


def _values(codes, params):
    """The values that codes [..., dim / 2] with (scale, zero) [..., 2] stand for, in 32 bits."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    params = params.float()
    return code * params[..., :1] + params[..., 1:]


def _load(pages, slots, block, dim):
    """Rows [tokens, kv_heads, dim] of the slots; zeros for negative slots."""
    codes, params = _parts(pages, block, dim)
    at, within = slots.clamp(min=0) // block, slots.clamp(min=0) % block
    rows = _values(codes[at, :, within], params[at, :, within])
    return torch.where((slots >= 0)[:, None, None], rows, torch.zeros_like(rows))


def _gathered(pages, tables, block, dim):
    """A tensor's values for each sequence, [batch, kv_heads, tokens, dim]."""
    codes, params = _parts(pages[tables.long()].transpose(1, 2), block, dim)
    return _values(codes, params).flatten(2, 3)


def _attend(s):
    query, lengths, device = s["query"], s["lengths"].long(), s["query"].device
    tokens, heads, dim = query.shape
    batch, most = lengths.shape[0], s["most"]
    key = _gathered(s["key_pages"], s["tables"], s["block"], dim)
    kv_heads, span = key.shape[1], key.shape[2]
    # Each sequence's query rows, padded to the longest.
    starts = s["starts"].long() if s["starts"] is not None else torch.arange(batch + 1, device=device) * most
    counts = starts[1:] - starts[:-1]
    at = torch.arange(most, device=device)
    real = at < counts[:, None]
    rows = torch.where(real, starts[:-1, None] + at, torch.zeros_like(starts[:-1, None] + at))
    q = query[rows].float().unflatten(2, (kv_heads, heads // kv_heads)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    score = torch.matmul(q, key.transpose(2, 3)).unflatten(2, (heads // kv_heads, most))
    del key
    score *= 1.0 / math.sqrt(dim)
    place = (lengths - counts)[:, None] + at
    j = torch.arange(span, device=device)
    seen = (j <= place[..., None]) & (place[..., None] < lengths[:, None, None])
    if s["window"]:
        seen &= (j > place[..., None] - s["window"]) | (j < s["sinks"])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    score -= top
    score.exp_()
    total = score.sum(-1, keepdim=True)
    value = _gathered(s["value_pages"], s["tables"], s["block"], dim)
    value = torch.where((j < lengths[:, None])[:, None, :, None], value, torch.zeros_like(value))
    out = torch.matmul(score.flatten(2, 3), value).unflatten(2, (heads // kv_heads, most))
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    lse = (top + total.log())[..., 0]
    full = torch.empty((tokens, heads, dim), device=device, dtype=query.dtype)
    full[rows[real]] = out.permute(0, 3, 1, 2, 4).flatten(2, 3)[real].to(query.dtype)
    full_lse = torch.empty((tokens, heads), device=device, dtype=torch.float32)
    full_lse[rows[real]] = lse.permute(0, 3, 1, 2).flatten(2, 3)[real]
    return full, full_lse


# ---- what a pass cannot do without ------------------------------------------------------------------------


def _pairs(case):
    """(query, key) pairs that attend, and cached tokens that some query of their sequence sees."""
    pairs = tokens = 0
    for n, m in zip(_lengths(case), _queries(case)):
        if not n:
            continue
        w, k = case["window"] or n, case["sinks"] if case["window"] else 0
        for p in range(n - m, n):
            low = max(0, p - w + 1)
            pairs += p + 1 - low + min(low, k) if p >= 0 else 0
        low = max(0, n - m - w + 1)
        tokens += n - low + min(low, k)
    return pairs, tokens


def work(case):
    row = case["head_dim"] // 2 + 4
    size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    if case["kind"] in ("write", "read"):
        rows = 2 * case["tokens"] * case["kv_heads"]
        real = 2 * (case["tokens"] - case.get("padded", 0)) * case["kv_heads"]
        wide = case["head_dim"] * size
        if case["kind"] == "read":
            return {"bytes": rows * (row + wide) + 8 * case["tokens"], "flops": 2 * rows * case["head_dim"]}
        # the rows are read, written as pages, and read back
        return {"bytes": real * (wide + 2 * row) + rows * wide + 8 * case["tokens"], "flops": 8 * real * case["head_dim"]}
    pairs, tokens = _pairs(case)
    asked = sum(_queries(case))
    moved = 2 * tokens * case["kv_heads"] * row + 2 * asked * case["heads"] * case["head_dim"] * size
    if case["lse"]:
        moved += 4 * asked * case["heads"]
    if case["kind"] == "turn":
        # the new rows: read, written as part of the pages, and given back
        moved += 2 * case["batch"] * case["kv_heads"] * (2 * case["head_dim"] * size + row)
    return {"bytes": moved, "flops": 4 * pairs * case["heads"] * case["head_dim"]}


# ---- the definition in 64 bits ----------------------------------------------------------------------------


def _exact_row(x):
    """What rows hold after they were written: x [..., dim] in 64 bits."""
    x = x.double().clamp(-LIMIT, LIMIT)
    low, high = torch.aminmax(x, dim=-1, keepdim=True)
    step, low = ((high - low) / 15).half().double(), low.half().double()
    n = torch.where(step > 0, (x - low) / torch.where(step > 0, step, torch.ones_like(step)), torch.zeros_like(x))
    return torch.round(n).clamp(0, 15) * step + low


def _exact_block(pages, block, dim):
    """Values [kv_heads, n * block, dim] of n pages [n, kv_heads, bytes]."""
    half = block * dim // 2
    packed = pages[:, :, :half].reshape(pages.shape[0], pages.shape[1], block, dim // 2)
    two = pages[:, :, half:].contiguous().view(torch.float16).reshape(pages.shape[0], pages.shape[1], block, 2).double()
    x = torch.empty((*packed.shape[:3], dim), device=pages.device, dtype=torch.float64)
    x[..., 0::2] = packed.remainder(16).double()
    x[..., 1::2] = packed.div(16, rounding_mode="floor").double()
    x = x * two[..., 0:1] + two[..., 1:2]
    return x.transpose(0, 1).reshape(pages.shape[1], -1, dim)


def exact(case, seed):
    s = prepare(case, seed)
    block, dim = case["block"], case["head_dim"]
    if case["kind"] == "write":
        live = (s["slots"] >= 0).double()[:, None, None]
        return {"key": _exact_row(s["key"]) * live, "value": _exact_row(s["value"]) * live}
    if case["kind"] == "read":
        got = {}
        for name in ("key", "value"):
            whole = _exact_block(s[name + "_pages"], block, dim)
            got[name] = whole[:, s["slots"]].transpose(0, 1).contiguous()
            del whole
        return got
    lengths, queries = _lengths(case), _queries(case)
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["query"].shape, device="cuda", dtype=torch.float64)
    lse = torch.full(s["query"].shape[:2], -math.inf, device="cuda", dtype=torch.float64)
    at = 0
    for i, (n, m) in enumerate(zip(lengths, queries)):
        if n:
            ids = s["tables"][i, : -(-n // block)].long()
            key, value = _exact_block(s["key_pages"][ids], block, dim)[:, :n], _exact_block(s["value_pages"][ids], block, dim)[:, :n]
            if case["kind"] == "turn":
                key[:, n - 1], value[:, n - 1] = _exact_row(s["key"][i]), _exact_row(s["value"][i])
            p = torch.arange(n - m, n, device="cuda")[:, None]
            j = torch.arange(n, device="cuda")[None]
            hidden = j > p
            if case["window"]:
                hidden |= (j <= p - case["window"]) & (j >= case["sinks"])
            for h in range(case["heads"]):
                x = s["query"][at:at + m, h].double() @ key[h // group].T / math.sqrt(dim)
                x = x.masked_fill(hidden, -math.inf)
                z = torch.logsumexp(x, -1, keepdim=True)
                none = torch.isinf(z)
                w = torch.exp(x - torch.where(none, torch.zeros_like(z), z))
                out[at:at + m, h] = w @ value[h // group]
                lse[at:at + m, h] = z[:, 0]
        at += m
    got = {"out": out, "lse": lse} if case["lse"] else {"out": out}
    if case["kind"] == "turn":
        live = (s["slots"] >= 0).double()[:, None, None]
        got.update(key=_exact_row(s["key"]) * live, value=_exact_row(s["value"]) * live)
    return got
