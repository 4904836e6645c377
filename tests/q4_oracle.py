"""The 4-bit paged cache in 64 bits, from its definition (test infrastructure)."""

import math

import torch

LIMIT = 65504.0


def quantise(x):
    """Rows x [..., dim] -> (codes uint8 [..., dim], scale fp16, zero fp16 [..., 1])."""
    x = x.detach().cpu().float()
    finite = torch.isfinite(x).all(-1, keepdim=True)
    c = torch.where(finite, x, torch.zeros_like(x)).clamp(-LIMIT, LIMIT)
    lo, hi = c.amin(-1, keepdim=True), c.amax(-1, keepdim=True)
    scale, zero = ((hi - lo) / 15).half(), lo.half()
    safe = torch.where(scale > 0, scale, torch.ones_like(scale)).double()
    codes = torch.round((c.double() - zero.double()) / safe).clamp(0, 15)
    codes = torch.where((scale > 0) & finite, codes, torch.zeros_like(codes)).to(torch.uint8)
    nan = torch.full_like(scale, math.nan)
    return codes, torch.where(finite, scale, nan), torch.where(finite, zero, nan)


def split(pages, dim):
    """Pages [blocks, heads, bytes] -> (codes [blocks, heads, P, dim], scale, zero [blocks, heads, P])."""
    pages = pages.detach().contiguous().cpu()
    block = pages.shape[-1] // (dim // 2 + 4)
    half = block * dim // 2
    packed = pages[..., :half].unflatten(-1, (block, dim // 2))
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)
    params = pages[..., half:].contiguous().view(torch.float16).unflatten(-1, (block, 2))
    return codes, params[..., 0], params[..., 1]


def values(pages, dim):
    """What pages stand for, float64 [blocks, heads, P, dim]."""
    codes, scale, zero = split(pages, dim)
    return codes.double() * scale.double()[..., None] + zero.double()[..., None]


def attention(query, key_pages, value_pages, tables, lens, starts=None, scale=None, window=None,
              sinks=0):
    """Attention by its definition, and how far a result computed as the kernels
    do may be from it: (out, lse, out_bound, lse_bound), float64.

    The bound's terms, for a row with weights p (sum 1):
      * its products q.c are summed in 32 bits in dim/16 steps and combined with
        three more roundings, each off by at most 2^-23 of the sum of the terms'
        magnitudes (an accumulation that truncates is off by a whole step), so a
        score is off by dx <= (dim/16 + 4) 2^-23 max_j sum_d |q_d| (s c_d + |z|) scale;
        exp2 of the hardware adds 2^-21.  Weights are off by that, relatively,
        and the normalised sum by twice that times the largest |v|;
      * each weight is rounded once to fp16 before the product with the codes:
        2^-11 of it, times |s (c - middle)| <= 8 s, since the middle of the codes
        (7.5 or 8) is taken off them;
      * sums in 32 bits: n/8 + 64 roundings of 2^-24, each of at most the largest
        |s c| + |z|; their middle part cancels at most twice;
      * the output is rounded to its type: half a step.
    """
    dim, group = query.shape[2], query.shape[1] // key_pages.shape[1]
    scale = 1 / math.sqrt(dim) if scale is None else scale
    tokens, heads = query.shape[:2]
    q = query.detach().double().cpu()
    k_codes, k_s, k_z = split(key_pages, dim)
    v_codes, v_s, v_z = split(value_pages, dim)
    block = k_codes.shape[2]
    lens, tables = lens.tolist(), tables.tolist()
    if starts is None:
        starts = [i * (tokens // max(1, len(lens))) for i in range(len(lens) + 1)]
    else:
        starts = starts.tolist()
    out = torch.zeros(tokens, heads, dim, dtype=torch.float64)
    lse = torch.full((tokens, heads), -math.inf, dtype=torch.float64)
    out_bound, lse_bound = torch.zeros_like(out), torch.zeros_like(lse)
    half = torch.finfo(query.dtype).eps / 2
    for b, n in enumerate(lens):
        rows = range(starts[b], starts[b + 1])
        if not len(rows):
            continue
        ids = tables[b][: -(-n // block)]
        at = lambda t: t[ids].transpose(0, 1).flatten(1, 2)[:, :n].double()  # noqa: E731
        kc, ks, kz, vc, vs, vz = (at(t) for t in (k_codes, k_s, k_z, v_codes, v_s, v_z))
        p = torch.arange(n - len(rows), n)[:, None]
        j = torch.arange(n)[None]
        seen = j <= p
        if window:
            seen &= (j > p - window) | (j < sinks)
        some = seen.any(1)
        for h in range(heads if n else 0):
            kv = h // group
            s, z, sv, zv = ks[kv][:, None], kz[kv][:, None], vs[kv], vz[kv]
            k, v = kc[kv] * s + z, vc[kv] * sv[:, None] + zv[:, None]
            x = q[rows.start:rows.stop, h] @ k.T * scale
            size = q[rows.start:rows.stop, h].abs() @ (kc[kv] * s + z.abs()).T * abs(scale)
            most = lambda t: torch.where(seen, t, torch.zeros(())).amax(1)  # noqa: E731
            dx = (dim / 16 + 4) * 2.0 ** -23 * most(size) + 2.0 ** -21
            x = torch.where(seen, x, -math.inf)
            total = torch.logsumexp(x, 1)
            w = torch.where(seen, torch.exp(x - total[:, None]), torch.zeros(()))
            w[~some] = 0
            o = w @ torch.where(seen.any(0)[:, None], v, torch.zeros(()))
            bound = 2 * dx * most(v.abs().amax(1)[None].expand_as(x))
            bound += 2.0 ** -11 * 8 * (w @ torch.where(seen.any(0), sv, torch.zeros(())))
            bound += 2 * (seen.sum(1) / 8 + 64) * 2.0 ** -24 * most((15 * sv + zv.abs())[None].expand_as(x))
            bound = bound[:, None]
            out[rows.start:rows.stop, h] = o
            lse[rows.start:rows.stop, h] = total
            out_bound[rows.start:rows.stop, h] = bound + half * (o.abs() + bound) + 2.0 ** -25
            lse_bound[rows.start:rows.stop, h] = dx + 2.0 ** -22 * (total.abs() + most(x.abs()) + 1)
    return out, lse, out_bound, lse_bound
